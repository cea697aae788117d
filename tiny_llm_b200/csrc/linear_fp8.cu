// 8-bit matrix products on the tensor cores:
//   C[m, n] = sum over groups g of 128 values of K:  sa[m, g] * sw[n / 128, g] * sum_{k in g} A[m, k] W[n, k]
// A [M, K] and W [N, K] are e4m3, sa one e8m0 scale per row and group, sw one float32 scale per block of 128 x 128.
//
// The products of a group are summed by the tensor cores in 32 bits (tcgen05.mma kind::f8f6f4, four instructions of K = 32) into one of the
// accumulators in tensor memory (two, or four for tiles of 128 columns).  While they fill the next one, the summing warps (sixteen; for few rows four
// to sixteen) read it back and add it, times the two scales, to 32-bit sums in registers: the scales of two groups differ, so the groups cannot be
// added up in tensor memory.  The sums are rounded once, when they leave:
//   * as bfloat16, as float32, or added to float32 rows;
//   * gated: the columns of a tile are 128 gate columns and the 128 matching up columns, act(gate) * up leaves as bfloat16 or in 8
//     bits again, with a scale per row and tile (its 128 columns are one group of the product behind it).
//
// Sizes: any M, N and K (up to FP8_MOST); rows of A and W start on 16 bytes.  TMA fills the tails with zeros, the epilogue masks them.  Every
// wait is bounded: on expiry the kernel records a code in `status`, stops issuing, frees its tensor memory and returns.
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "fp8.cuh"
#include "fp8_calls.h"
#include "tc_common.cuh"

TLLM_DEFINE_LAST_ERROR

namespace tllm {

constexpr int BM = 128;          // rows of A per CTA = MMA M
constexpr int BK = FP8_GROUP;    // values of K per stage: one group, one 128-byte swizzle row
constexpr int UMMA_K = 32;
constexpr int SUM_WARPS = 16;    // warps that scale and add: four per 32 rows, a quarter of the columns each
constexpr int FIRST_SUM_WARP = 4;  // warp 0: TMA, warp 1: MMA + tensor-memory allocation, 2 and 3 fill the warpgroup
constexpr int THREADS = 32 * (FIRST_SUM_WARP + SUM_WARPS);
// Registers: the launch gives 96 to each of 640 threads; the first warpgroup hands most of its own to the four that sum
// (128 * 32 + 512 * 112 = 640 * 96).
constexpr int REGS_OTHERS = 32, REGS_SUMS = 112;
constexpr int STAGING_BYTES = 16 * 32 * 4;     // of shared memory per summing warp, for its stores
constexpr int BAND = 12;         // row tiles per band of the large products' order

enum Output { OUT_BF16 = 0, OUT_F32 = 1, OUT_ADD = 2, OUT_FP8 = 3 };
enum Act { ACT_SILU = 0, ACT_RELU = 1, ACT_CLAMPED = 2, ACT_GELU_TANH = 3 };

// act(g) * u for all four gates without a branch (the code is laid out 32 times per thread): with g and u clamped,
// g / (1 + exp(-g (a + b g^2) - e)) * (u + d).  SiLU: a = 1; GELU's tanh form z / 2 (1 + tanh(y)) = z / (1 + exp(-2 y)): a = 2 sqrt(2 / pi),
// b = 0.044715 a; clamped: a = 1.702, d = 1; ReLU: g from 0 on, a = 0, and exp(-e) is 0, so that g is what is left.
struct Gate { float g_low, g_high, u_most, a, b, d, e; };
static Gate make_gate(int act, float limit) {
  const float inf = INFINITY;
  if (act == ACT_RELU) return {0.f, inf, inf, 0.f, 0.f, 0.f, 200.f};
  if (act == ACT_CLAMPED) return {-inf, limit, limit, 1.702f, 0.f, 1.f, 0.f};
  if (act == ACT_GELU_TANH) return {-inf, inf, inf, 1.59576912160573081f, 1.59576912160573081f * 0.044715f, 0.f, 0.f};
  return {-inf, inf, inf, 1.f, 0.f, 0.f, 0.f};
}
struct Fp8Args {
  const uint8_t *a, *w;        // e4m3 rows, for the sums made once more (the products read them through the copy unit)
  const uint8_t* a_scales;     // [m][lda_s] e8m0
  const float* w_scales;       // [ceil(n / 128)][groups]
  void* out;
  uint8_t* out_scales;         // OUT_FP8: [m][ldo_s] e8m0
  long long lda, ldw, lda_s, ldo, ldo_s;
  int m, n, k, w_rows, groups;            // n: columns of `out` (gated: half the weight's rows, without the ones that fill the last block)
  int mode;
  int vec_out;                 // rows of `out` start on 16 bytes
  int vec_scales;              // rows of a_scales start on 4 bytes
  Gate gate;
};

// (a NaN stays one)
__device__ __forceinline__ float max_nan(float x, float y) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float min_nan(float x, float y) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float gate_f(float g, float u, const Gate& q) {
  g = min_nan(max_nan(g, q.g_low), q.g_high);
  u = min_nan(max_nan(u, -q.u_most), q.u_most);
  // With x = exp(-|argument|), at most 1: g / (1 + x) from zero on and g x / (1 + x) below, so that nothing leaves 32 bits before the
  // result does.  The quotient to half a unit: an approximate reciprocal of a number from 1 to 2 and one step with the exact remainder;
  // where the result is rounded to 8 bits, every unit moves values across borders.
  // An infinite sum stays infinite: the argument is taken at 1e15, where every gate has long been its input, and the remainder of an
  // infinity, a NaN, is dropped; below zero the gate is 0 there.
  const float h = min_nan(max_nan(g, -1e15f), 1e15f), x = expf(fmaf(-fabsf(h), fmaf(q.b * h, h, q.a), -q.e));
  const float n = h < 0.f ? h * x : g, d = 1.f + x;
  const float r = __fdividef(1.f, d), y = n * r;
  return fmaf(fmaxf(fmaf(-y, d, n), -FLT_MAX), r, y) * (u + q.d);
}

// A group's sum meets the product of two scales, which may lie anywhere in 32 bits: the product may leave them although the result does not
// (2^100 * 2^40 beside a sum of 0 or 2^-18), or keep few bits below 2^-126.  The kernels note such products, and the elements they belong to are
// summed once more, one by one and in 64 bits.  The scales of a model's rows and weights lie within a few powers of ten, so this is for
// being right and not for speed: with such a product in each row, 8 rows of 4,096 x 14,336 take 6 ms and 2,048 rows 70 (20 per tile; the
// CTA's other warps wait for 2 s, which a K of a million and a half would use up, as the status word then says).  The way of all others
// pays an instruction or two per product for it (1 x 2,560 x 2,048 3.08 us -> 3.12, 64 x 5,632 x 2,048 gated 10.3 -> 10.6, many rows at most
// 2 %).  Two factors in place of the product, applied one after the other, cost every call 2 to 7 %.
__device__ __forceinline__ uint32_t far_key(float s) { return 2u * __float_as_uint(s) - 0x01000000u; }      // FAR or more unless s is a normal number
constexpr uint32_t FAR = 0xFE000000u;
// (zeros, infinities and NaN among the scales themselves give what they give)
__device__ __forceinline__ bool is_far(uint32_t byte, float w) { return far_key(fp8_scale(byte) * w) >= FAR && byte != 255u && w != 0.f && isfinite(w); }
__device__ __forceinline__ float far_sum(const Fp8Args& p, int m, int w_row) {
  const uint8_t *a = p.a + m * p.lda, *w = p.w + w_row * p.ldw, *sa = p.a_scales + m * p.lda_s;
  const float* sw = p.w_scales + (long long)(w_row / 128) * p.groups;
  auto value = [](uint8_t v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3))); };
  double sum = 0.;
  for (int g = 0; g < p.groups; ++g) {
    double part = 0.;
    const int end = min(p.k, (g + 1) * BK);
#pragma unroll 1
    for (int k = g * BK; k < end; ++k) part += value(a[k]) * value(w[k]);       // (a product of two has 8 bits)
    sum += part * fp8_scale(sa[g]) * sw[g];
  }
  return (float)sum;
}

// sixteen values of a row from `k` on, zeros behind its last
__device__ __forceinline__ void load16(const uint8_t* row, int k, int width, float* v) {
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if (k + 16 <= width) {
    u = *reinterpret_cast<const uint4*>(row + k);
  } else {
    for (int e = 0; k + e < width; ++e) (&u.x)[e / 4] |= (uint32_t)row[k + e] << (8 * (e % 4));
  }
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((&u.x)[e / 4] >> (8 * (e % 4))), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[e] = f.x; v[e + 1] = f.y;
  }
}
// The same for 32 neighbouring rows of the weight, 0 behind the last one (what a thread of the large tiles has): sixteen products at a time in 32
// bits, five roundings each at most, scaled and added up in 64.
__device__ __noinline__ void far_sums(const Fp8Args& p, int m, int w_row, float* again) {
  double sums[32];
#pragma unroll 1
  for (int j = 0; j < 32; ++j) sums[j] = 0.;
  const uint8_t *a = p.a + m * p.lda, *sa = p.a_scales + m * p.lda_s;
#pragma unroll 1
  for (int k = 0; k < p.k; k += 16) {
    const int g = k / BK;
    const double scale = fp8_scale(sa[g]);
    float x[16];
    load16(a, k, p.k, x);
#pragma unroll 1
    for (int j = 0; j < 32; ++j) {
      const int row = w_row + j;
      if (row >= p.w_rows) break;
      float y[16], part[4] = {0.f, 0.f, 0.f, 0.f};
      load16(p.w + row * p.ldw, k, p.k, y);
#pragma unroll
      for (int e = 0; e < 16; ++e) part[e % 4] = fmaf(x[e], y[e], part[e % 4]);
      sums[j] += (double)((part[0] + part[1]) + (part[2] + part[3])) * (scale * p.w_scales[(long long)(row / 128) * p.groups + g]);
    }
  }
#pragma unroll 1
  for (int j = 0; j < 32; ++j) again[j] = (float)sums[j];
}

// e4m3 x e4m3 -> float32, M = m, N = n, both operands K-major (bits 7-9 and 10-12: 0 is e4m3)
__device__ __forceinline__ uint32_t instr_desc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void umma_fp8_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(SMEM_DESC_SW128_HI) : "memory");
}
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
// Waits for this warp's loads from tensor memory; naming the registers keeps the arithmetic on them behind the wait.
__device__ __forceinline__ void tmem_ld32_arrived(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
// (c0, c1) + (a0, a1) * s in one instruction
__device__ __forceinline__ float2 fma2(uint32_t a0, uint32_t a1, float2 s, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "r"(a0), "r"(a1), "f"(s.x), "f"(s.y), "f"(c.x), "f"(c.y));
  return r;
}
// true in all the summing warps only if `ok` holds in all of them
__device__ __forceinline__ bool sums_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "r"((uint32_t)ok), "n"(32 * SUM_WARPS) : "memory");
  return r != 0;
}
// ---- a cluster of CTAs: where `p` of this CTA lies in the CTA of that rank, and a store there that its barrier counts
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void st_async_f32(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}
// (Relaxed: what the peers have to see is the barriers' initial state, which has a fence of its own, and sums, which are counted by a
// barrier; a release here is a fence over all memory, 0.3 us each time.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

template <int BN, int STAGES>
struct Smem {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGING_OFFSET = STAGES * STAGE_BYTES;        // what the summing warps store passes here, or the largest magnitudes
  static constexpr int BAR_OFFSET = STAGING_OFFSET + SUM_WARPS * STAGING_BYTES;                                      // of a row's four parts
  static constexpr int ACCS = 512 / BN;            // accumulators in tensor memory: the products run that many groups ahead of the sums
  static constexpr int TOTAL = BAR_OFFSET + (2 * STAGES + 2 * ACCS) * 8 + 16 + 1024;
};

// eight columns as bfloat16
__device__ __forceinline__ uint4 pack8_bf16(float4 a, float4 b) {
  uint4 pk;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&pk);
  h[0] = __floats2bfloat162_rn(a.x, a.y); h[1] = __floats2bfloat162_rn(a.z, a.w);
  h[2] = __floats2bfloat162_rn(b.x, b.y); h[3] = __floats2bfloat162_rn(b.z, b.w);
  return pk;
}

// A warp's 32 rows (lane l has row m0 + l) of 32 columns from `n` on leave as `mode` says.  They pass through 2 KB of the warp's own in
// shared memory, 16 rows at a time, so that a store of the warp covers 64 or 128 neighbouring bytes of few rows: straight from the
// registers every store touched 32 rows, and with rows that do not start on 16 bytes, value by value, that took longer than the products
// (8,192 rows of 300 x 4,096: 56 us).
__device__ __forceinline__ void store_columns(const Fp8Args& p, float* staging, int m0, int n, const float* v, int mode) {
  const int lane = threadIdx.x & 31;
  const bool vec = p.vec_out && n + 32 <= p.n;
  // 16 bytes c of row r lie at place c ^ (r % 8) of the row's eight
  auto place = [&](int r, int c) { return reinterpret_cast<float4*>(staging + r * 32) + (c ^ (r & 7)); };
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 16) {
    __syncwarp();
    if ((lane & 16) == r0) {
#pragma unroll
      for (int c = 0; c < 8; ++c) *place(lane & 15, c) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    }
    __syncwarp();
    if (vec && mode == OUT_BF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * i + lane / 4, c = lane % 4, m = m0 + r0 + r;
        const uint4 pk = pack8_bf16(*place(r, 2 * c), *place(r, 2 * c + 1));
        if (m < p.m) *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + (size_t)m * p.ldo + n + 8 * c) = pk;
      }
    } else if (vec) {
      float4 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + r0 + 4 * i + lane / 8;
        if (mode == OUT_ADD && m < p.m) o[i] = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n + 4 * (lane % 8));
        else o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + lane / 8, m = m0 + r0 + r;
        const float4 x = *place(r, lane % 8);
        o[i].x += x.x; o[i].y += x.y; o[i].z += x.z; o[i].w += x.w;
        if (m < p.m) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n + 4 * (lane % 8)) = o[i];
      }
    } else {
#pragma unroll 4
      for (int r = 0; r < 16; ++r) {
        const int m = m0 + r0 + r;
        const float x = reinterpret_cast<float*>(place(r, lane / 4))[lane % 4];
        if (m < p.m && n + lane < p.n) {
          const size_t at = (size_t)m * p.ldo + n + lane;
          if (mode == OUT_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
          else if (mode == OUT_ADD) reinterpret_cast<float*>(p.out)[at] += x;
          else reinterpret_cast<float*>(p.out)[at] = x;
        }
      }
    }
  }
}

template <int BN, int STAGES, bool GATED>
__global__ void __launch_bounds__(THREADS, 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Fp8Args p, int* __restrict__ status) {
  static_assert(!GATED || BN == 256, "a gated tile is one group of gate columns and one of up columns");
  using L = Smem<BN, STAGES>;
  constexpr int ACCS = L::ACCS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint32_t* most = reinterpret_cast<uint32_t*>(smem + L::STAGING_OFFSET);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::BAR_OFFSET);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;      // accumulator b holds a group's products
  uint64_t* acc_empty = acc_full + ACCS;        // the summing warps have read accumulator b
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + ACCS);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (p.m + BM - 1) / BM, tiles_n = GATED ? (p.n + 127) / 128 : (p.n + BN - 1) / BN;
  const int n_tiles = tiles_m * tiles_n;

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_a); tma_prefetch_map(&map_w);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < ACCS; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], SUM_WARPS); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  // Tile t: the row tiles in bands of BAND, inside a band the row tiles of one column of tiles are neighbours.  The tiles that run side
  // by side then share both operands: about 12 x 12 of them instead of all row tiles by two or three columns.
  auto tile_at = [&](int t, int& tm, int& tn) {
    const int band = t / (BAND * tiles_n), first = band * BAND, high = min(BAND, tiles_m - first), in = t - band * BAND * tiles_n;
    tm = first + in % high;
    tn = in / high;
  };

  if (warp < FIRST_SUM_WARP) {
    regs_down<REGS_OTHERS>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x) {
        int tm, tn;
        tile_at(t, tm, tn);
        for (int g = 0; g < p.groups; ++g, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { *abort_flag = 1; atomicExch(status, ERR_QP_PRODUCER); ok = false; break; }
          uint8_t* dst = smem + s * L::STAGE_BYTES;
          mbar_expect_tx(&full_bar[s], L::STAGE_BYTES);
          tma_load_2d(dst, &map_a, g * BK, tm * BM, &full_bar[s]);
          tma_load_2d(dst + L::A_BYTES, &map_w, g * BK, tn * BN, &full_bar[s]);
        }
      }
      mbar_drain(full_bar, STAGES, it);
    } else if (warp == 1) {
      // ---------------- MMA issuer (warp-wide loop, one elected lane issues)
      const uint32_t idesc = instr_desc_e4m3(BM, BN);
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint32_t lo0 = smem_desc_sw128_lo(smem_u32(smem));
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x)
        for (int g = 0; g < p.groups; ++g, ++it) {
          const int s = it % STAGES, buf = it % ACCS;
          ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((it / ACCS) & 1) ^ 1, abort_flag) && mbar_wait(&full_bar[s], (it / STAGES) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = lo0 + s * (L::STAGE_BYTES >> 4), b_lo = a_lo + (L::A_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k)
              umma_fp8_lo(tmem_u + buf * BN, a_lo + (k * UMMA_K >> 4), b_lo + (k * UMMA_K >> 4), idesc, k > 0 ? 1u : 0u);
            umma_commit(&empty_bar[s]);
            umma_commit(&acc_full[buf]);
          }
          __syncwarp();
        }
      if (!ok && lane == 0) { *abort_flag = 1; atomicExch(status, ERR_QP_MMA); }
    }
  } else {
    regs_up<REGS_SUMS>();
    // ---------------- sums: warp w reads tensor-memory lanes [32 (w % 4), +32), and of its row a quarter of the columns: with a
    // plain tile [part * BN / 4, +BN / 4), with a gated one 32 gate columns and the 32 matching up columns
    constexpr int COLS = BN / 4, CHUNKS = COLS / 32;
    const int quad = warp & 3, part = (warp - FIRST_SUM_WARP) >> 2;
    const int row = quad * 32 + lane;
    float* staging = reinterpret_cast<float*>(smem + L::STAGING_OFFSET) + (warp - FIRST_SUM_WARP) * (STAGING_BYTES / 4);
    auto column = [&](int c) { return GATED ? part * 32 + 128 * c : part * COLS + 32 * c; };
    int it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < n_tiles; t += gridDim.x) {
      int tm, tile_n;
      tile_at(t, tm, tile_n);
      const int m = tm * BM + row;
      // the row's scales, four groups to a word where the rows allow it
      const uint8_t* sa = p.a_scales + (long long)min(m, p.m - 1) * p.lda_s;
      auto four_scales = [&](int g) -> uint32_t {
        if (g >= p.groups) return 0u;
        if (p.vec_scales && g + 4 <= p.groups) return *reinterpret_cast<const uint32_t*>(sa + g);
        uint32_t q = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (g + e < p.groups) q |= (uint32_t)sa[g + e] << (8 * e);
        return q;
      };
      // the rows of W that a thread reads lie in one block of 128 (gated: one of gate, one of up), the last one where W ends inside a tile
      const int block = GATED ? 2 * tile_n : min((tile_n * BN + part * COLS) / 128, (p.n - 1) / 128);
      const float* sw = p.w_scales + (long long)block * p.groups;
      float acc[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
      uint32_t quad_now = 0u, quad_next = four_scales(0);
      float w0 = sw[0], w1 = GATED ? sw[p.groups] : 0.f;
      uint32_t farthest = 0u;
      for (int g = 0; g < p.groups; ++g, ++it) {
        const int buf = it % ACCS;
        if ((g & 3) == 0) { quad_now = quad_next; quad_next = four_scales(g + 4); }
        const float a = fp8_scale((quad_now >> (8 * (g & 3))) & 255u), s0 = a * w0, s1 = a * w1;
        farthest = max(farthest, GATED ? max(far_key(s0), far_key(s1)) : far_key(s0));
        if (g + 1 < p.groups) { w0 = sw[g + 1]; if (GATED) w1 = sw[p.groups + g + 1]; }
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (it / ACCS) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + buf * BN + ((uint32_t)(quad * 32) << 16);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          uint32_t v[32];
          tmem_ld32_issue(taddr + column(c), v);
          tmem_ld32_arrived(v);
          if (c == CHUNKS - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
          }
          const float s = GATED && c > 0 ? s1 : s0;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 r = fma2(v[j], v[j + 1], make_float2(s, s), make_float2(acc[32 * c + j], acc[32 * c + j + 1]));
            acc[32 * c + j] = r.x;
            acc[32 * c + j + 1] = r.y;
          }
        }
      }
      if (!ok && lane == 0) { *abort_flag = 1; atomicExch(status, ERR_QP_SUMS); }
      if (!sums_all(ok)) break;
      if (__builtin_expect(__any_sync(0xffffffffu, farthest >= FAR), 0)) {
        bool far = false;
        if (farthest >= FAR && m < p.m)
          for (int g = 0; g < p.groups; ++g) far = far || is_far(sa[g], sw[g]) || (GATED && is_far(sa[g], sw[p.groups + g]));
        // (all sums pass through memory, so that none is held in a register over the calls: held, they cost the loop above a quarter)
        float again[COLS];
#pragma unroll
        for (int j = 0; j < COLS; ++j) again[j] = acc[j];
        if (far) {
#pragma unroll 1
          for (int c = 0; c < CHUNKS; ++c) far_sums(p, m, tile_n * BN + column(c), again + 32 * c);
        }
#pragma unroll
        for (int j = 0; j < COLS; ++j) acc[j] = again[j];
        __syncwarp();
      }
      if (!GATED) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) store_columns(p, staging, m - lane, tile_n * BN + column(c), acc + 32 * c, p.mode);
      } else {
        const int n = tile_n * 128 + part * 32;
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[j] = n + j < p.n ? gate_f(acc[j], acc[32 + j], p.gate) : 0.f;
        if (p.mode != OUT_FP8) {
          store_columns(p, staging, m - lane, n, acc, OUT_BF16);
        } else {
          uint32_t largest = 0u;
#pragma unroll
          for (int j = 0; j < 32; ++j) largest = max(largest, fp8_abs_bits(acc[j]));
          most[part * BM + row] = largest;
          sums_all(true);
          const uint32_t byte = fp8_scale_byte(max(max(most[row], most[BM + row]), max(most[2 * BM + row], most[3 * BM + row])));
          const float inverse = fp8_inverse_scale(byte);
          if (m < p.m) {
            uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + (size_t)m * p.ldo + n;
            if (part == 0) p.out_scales[(size_t)m * p.ldo_s + tile_n] = (uint8_t)byte;
#pragma unroll
            for (int j = 0; j < 32; j += 16) {
              uint4 pk;
              pk.x = fp8_pack4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3], inverse, byte);
              pk.y = fp8_pack4(acc[j + 4], acc[j + 5], acc[j + 6], acc[j + 7], inverse, byte);
              pk.z = fp8_pack4(acc[j + 8], acc[j + 9], acc[j + 10], acc[j + 11], inverse, byte);
              pk.w = fp8_pack4(acc[j + 12], acc[j + 13], acc[j + 14], acc[j + 15], inverse, byte);
              if (n + j + 16 <= p.n) {
                *reinterpret_cast<uint4*>(dst + j) = pk;
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  if (n + j + e < p.n) dst[j + e] = (uint8_t)((&pk.x)[e / 4] >> (8 * (e % 4)));
              }
            }
          }
          sums_all(true);   // the next tile's largest magnitudes wait for this one's readers
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------- few rows
// The weight is the 128-row operand, up to 128 rows of A are the BN columns of a tile, and K is cut into slices so that every SM streams
// weights (more rows of A are more tiles, which fetch the weight again; see pick_kernel); such a product is bound by reading them once, and short ones by the way from the last product to the last store.
// The slices of one tile are a thread-block cluster, and token j of the tile belongs to CTA j % slices of it.  Every CTA adds its groups
// up in registers (a thread per weight row) and sends each token's sums to the CTA it belongs to (st.async, counted by a barrier there);
// that one adds the slices in a fixed order, a warp per token, four weight rows per lane, and stores 128 neighbouring columns.  No CTA
// waits for the cluster: sums that the owner reads from the others between two cluster barriers took 3,300 cycles from the last sum to
// the end of the kernel, of 6,100 for one row of 2,560 x 2,048.  Gated: a CTA has the gate tile and the up tile beside it, two
// accumulators and four warps for each; the 128 columns that a warp stores are one group of the product behind.
// A tile's columns are dealt to HALVES sets of four summing warps.
template <int BN, int STAGES, bool GATED, int HALVES, bool SLICED, int SENT = BN + 8>
struct FewSmem {
  static constexpr int SUM_WARPS = 4 * (GATED ? 2 : 1) * HALVES, THREADS = 64 + 32 * SUM_WARPS;
  static constexpr int CHUNK = BN >= 64 || GATED ? 4 : 8;                      // groups whose scales are laid out in shared memory at a time
  static constexpr int TILES = GATED ? 2 : 1, W_BYTES = TILES * 128 * BK, A_BYTES = BN * BK, STAGE_BYTES = W_BYTES + A_BYTES;
  // The sums: [tokens of this CTA][slices][TILES][128 weight rows].  The peers may send theirs while this CTA still works, so they have a
  // place of their own, of SENT = tokens per CTA x slices (at most 7 more than BN); a CTA without peers leaves them where the stages were.
  static constexpr int SUMS_OFFSET = SLICED ? STAGES * STAGE_BYTES : 0;
  static constexpr int SCALE_OFFSET = STAGES * STAGE_BYTES + (SLICED ? SENT * TILES * 512 : 0);
  static constexpr int BAR_OFFSET = SCALE_OFFSET + TILES * CHUNK * BN * 4;
  static constexpr int TOTAL = BAR_OFFSET + (2 * STAGES + 5) * 8 + 16 + 1024;
  static constexpr int RESIDENT = TOTAL <= 113 * 1024 && THREADS <= 320 ? 2 : 1;     // CTAs per SM
  static_assert(!(GATED && BN == 16) || RESIDENT == 2, "two CTAs per SM");
  static_assert(SLICED || TILES * BN * 512 <= STAGES * STAGE_BYTES, "the sums fit where the stages were");
};

struct FewArgs {
  int slices, per_slice;       // slices of K (the cluster), groups per slice (the last may have fewer, or none)
};

template <int BN, int STAGES, bool GATED, int HALVES, bool SLICED, int SENT = BN + 8>
__global__ void __launch_bounds__(FewSmem<BN, STAGES, GATED, HALVES, SLICED, SENT>::THREADS, FewSmem<BN, STAGES, GATED, HALVES, SLICED, SENT>::RESIDENT)
linear_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Fp8Args p, const FewArgs f, int* __restrict__ status) {
  using L = FewSmem<BN, STAGES, GATED, HALVES, SLICED, SENT>;
  constexpr int FEW_CHUNK = L::CHUNK, TILES = L::TILES, FEW_SUM_WARPS = L::SUM_WARPS, WARPS = 2 + FEW_SUM_WARPS;
  constexpr uint32_t ACC_COLS = TILES * BN, TMEM_COLS = 2 * ACC_COLS < 32 ? 32 : 2 * ACC_COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* scale = reinterpret_cast<float*>(smem + L::SCALE_OFFSET);     // [TILES][FEW_CHUNK][BN]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::BAR_OFFSET);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* sums_bar = acc_empty + 2;           // the slices' sums of this CTA's tokens are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_bar + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* sums = reinterpret_cast<float*>(smem + L::SUMS_OFFSET);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * BN, tile = blockIdx.y, rank = blockIdx.z;
  const int g_begin = min(p.groups, rank * f.per_slice), n_g = min(p.groups, g_begin + f.per_slice) - g_begin;
  const int tokens = min(BN, p.m - m0), own_tokens = tokens > rank ? (tokens - rank + f.slices - 1) / f.slices : 0;

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_w); tma_prefetch_map(&map_a);
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], FEW_SUM_WARPS); }
    mbar_init(sums_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (SLICED) mbar_expect_tx(sums_bar, own_tokens * f.slices * TILES * 512);
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (SLICED) cluster_arrive();        // (waited for below, when everybody has long been here: the peers' barriers are there to be counted on)
  // the weight depends on no earlier kernel: the first stages are asked for before this grid waits for its predecessors
  pdl_trigger();
  const int n_pre = min(n_g, STAGES);
  auto load_weight = [&](int i, uint64_t policy) {
    const int s = i % STAGES;
    mbar_expect_tx(&full_bar[s], L::STAGE_BYTES);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      tma_load_2d_hint(smem + s * L::STAGE_BYTES + t * 128 * BK, &map_w, (g_begin + i) * BK, (tile * TILES + t) * 128, &full_bar[s], policy);
  };
  // (A weight that one tile of rows reads is read once.  Where several share it the hint does no harm either, they run at the same time: us with it /
  // without, 64 rows of 2,560 x 2,048 4.76 / 4.85, 128 6.0 / 6.2, 64 of 4,096 x 4,096 7.1 / 7.3, 300 of 2,000 x 4,000 12.2 / 12.5.)
  const uint64_t policy = l2_evict_first_policy();
  if (warp == 0 && lane == 0)
    for (int i = 0; i < n_pre; ++i) load_weight(i, policy);
  pdl_wait();
  if (SLICED) cluster_wait();
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer
      int i = 0;
      for (; i < n_g; ++i) {
        const int s = i % STAGES;
        if (i >= n_pre) {
          if (!mbar_wait(&empty_bar[s], ((i / STAGES) & 1) ^ 1, abort_flag)) { *abort_flag = 1; atomicExch(status, ERR_QP_PRODUCER); break; }
          load_weight(i, policy);
        }
        tma_load_2d(smem + s * L::STAGE_BYTES + L::W_BYTES, &map_a, (g_begin + i) * BK, m0, &full_bar[s]);
      }
      mbar_drain(full_bar, STAGES, i);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer
    const uint32_t idesc = instr_desc_e4m3(128, BN);
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint32_t lo0 = smem_desc_sw128_lo(smem_u32(smem));
    for (int i = 0; i < n_g; ++i) {
      const int s = i % STAGES, buf = i & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((i >> 1) & 1) ^ 1, abort_flag) && mbar_wait(&full_bar[s], (i / STAGES) & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint32_t w_lo = lo0 + s * (L::STAGE_BYTES >> 4), a_lo = w_lo + (L::W_BYTES >> 4);
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_fp8_lo(tmem_u + buf * ACC_COLS + t * BN, w_lo + (t * 128 * BK >> 4) + (k * UMMA_K >> 4), a_lo + (k * UMMA_K >> 4), idesc, k > 0 ? 1u : 0u);
        umma_commit(&empty_bar[s]);
        umma_commit(&acc_full[buf]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) { *abort_flag = 1; atomicExch(status, ERR_QP_MMA); }
  } else {
    // ---------------- sums: warp w reads tensor-memory lanes [32 (w % 4), +32) of its tile's accumulator, COLS columns of it
    constexpr int COLS = BN / HALVES;
    const int quad = warp & 3, set = (warp - 2) >> 2, part = set / HALVES, col0 = (set % HALVES) * COLS, thread = threadIdx.x - 64;
    const int row = quad * 32 + lane;
    float acc[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
    // the scales of a chunk of groups: fetched while the chunk before is added up, the row's times the block's in shared memory
    constexpr int FETCH = (FEW_CHUNK * BN + 32 * FEW_SUM_WARPS - 1) / (32 * FEW_SUM_WARPS);
    float fetched[FETCH][TILES];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int q = 0; q < FETCH; ++q) {
        const int e = thread + q * 32 * FEW_SUM_WARPS, g = e % FEW_CHUNK, j = e / FEW_CHUNK;
        const bool there = j < BN && i0 + g < n_g && m0 + j < p.m;
        const float a = there ? fp8_scale(p.a_scales[(long long)(m0 + j) * p.lda_s + g_begin + i0 + g]) : 1.f;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const float s = there ? a * p.w_scales[(long long)(tile * TILES + t) * p.groups + g_begin + i0 + g] : 1.f;
          fetched[q][t] = far_key(s) >= FAR ? __uint_as_float(0x7FC00000u) : s;      // (the token's owner sees the NaN)
        }
      }
    };
    fetch(0);
    for (int i0 = 0; i0 < n_g; i0 += FEW_CHUNK) {
      const int n = min(FEW_CHUNK, n_g - i0);
      asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_SUM_WARPS) : "memory");     // the chunk before has been read
#pragma unroll
      for (int q = 0; q < FETCH; ++q) {
        const int e = thread + q * 32 * FEW_SUM_WARPS, g = e % FEW_CHUNK, j = e / FEW_CHUNK;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          if (j < BN) scale[(t * FEW_CHUNK + g) * BN + j] = fetched[q][t];
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_SUM_WARPS) : "memory");
      if (i0 + FEW_CHUNK < n_g) fetch(i0 + FEW_CHUNK);
      for (int g = 0; g < n && ok; ++g) {
        const int i = i0 + g, buf = i & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (i >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + buf * ACC_COLS + part * BN + col0 + ((uint32_t)(quad * 32) << 16);
        const float4* sc = reinterpret_cast<const float4*>(scale + (part * FEW_CHUNK + g) * BN + col0);
        auto add = [&](float* to, const uint32_t* v, int c) {      // four columns
          const float4 s4 = sc[c / 4];
          const float2 lo = fma2(v[0], v[1], make_float2(s4.x, s4.y), make_float2(to[0], to[1]));
          const float2 hi = fma2(v[2], v[3], make_float2(s4.z, s4.w), make_float2(to[2], to[3]));
          to[0] = lo.x; to[1] = lo.y; to[2] = hi.x; to[3] = hi.y;
        };
        if constexpr (COLS == 16) {
          float v[16];
          tmem_ld16(taddr, v);
#pragma unroll
          for (int j = 0; j < 16; j += 4) add(acc + j, reinterpret_cast<const uint32_t*>(v) + j, j);
        } else {
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            uint32_t v[32];
            tmem_ld32_issue(taddr + c, v);
            tmem_ld32_arrived(v);
#pragma unroll
            for (int j = 0; j < 32; j += 4) add(acc + c + j, v + j, c + j);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
    }
    if (!ok && lane == 0) { *abort_flag = 1; atomicExch(status, ERR_QP_SUMS); }
    int owner = col0 % f.slices, place = col0 / f.slices;
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (!SLICED) {      // the last accumulator is there, so every product has read its stage: the stages are free
        sums[((col0 + j) * TILES + part) * 128 + row] = acc[j];
        continue;
      }
      if (col0 + j < tokens)
        st_async_f32(cluster_addr(sums + ((place * f.slices + rank) * TILES + part) * 128 + row, owner), acc[j], cluster_addr(sums_bar, owner));
      if (++owner == f.slices) { owner = 0; ++place; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);

  if (SLICED) cluster_arrive();        // this CTA has sent what it had to
  // (one answer for the warp: what follows has steps that all its lanes take together)
  const bool here = __all_sync(0xffffffffu, !SLICED || own_tokens == 0 || mbar_wait(sums_bar, 0, abort_flag));
  if (!here && lane == 0) { *abort_flag = 1; atomicExch(status, ERR_QP_SUMS); }
  // Token i of this CTA.  A sum is NaN by scales whose product is no normal number, or by a row's own (or a weight's): such tokens come a second
  // time, with those sums made one by one (a row with a scale that is NaN stays NaN).  Returns whether the lane has met a NaN.
  auto leave = [&](int i, auto is_far) -> bool {
    constexpr bool FAR_SUMS = decltype(is_far)::value;
    const int m = m0 + rank + i * f.slices, n = tile * 128 + 4 * lane;
    float4 part[TILES][8];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (SLICED ? z < f.slices : z == 0) part[t][z] = reinterpret_cast<const float4*>(sums)[((i * f.slices + z) * TILES + t) * 32 + lane];
    float sum[TILES][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      sum[t][0] = sum[t][1] = sum[t][2] = sum[t][3] = 0.f;
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (SLICED ? z < f.slices : z == 0) { sum[t][0] += part[t][z].x; sum[t][1] += part[t][z].y; sum[t][2] += part[t][z].z; sum[t][3] += part[t][z].w; }
    }
    bool nan = (FAR_SUMS || !GATED) && isnan((sum[0][0] + sum[0][1]) + (sum[0][2] + sum[0][3]));
    if constexpr (FAR_SUMS) {
      if (GATED) nan = nan || isnan((sum[TILES - 1][0] + sum[TILES - 1][1]) + (sum[TILES - 1][2] + sum[TILES - 1][3]));
      if (!__any_sync(0xffffffffu, nan)) return false;
      bool nan_row = false;
      for (int g = 0; g < p.groups; ++g) nan_row = nan_row || p.a_scales[m * p.lda_s + g] == 255;
      if (nan && !nan_row) {
        float again[4 * TILES];
#pragma unroll 1
        for (int j = 0; j < 4 * TILES; ++j) {
          const int w_row = (tile * TILES + j / 4) * 128 + 4 * lane + j % 4;
          again[j] = w_row < p.w_rows ? far_sum(p, m, w_row) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4 * TILES; ++j) sum[j / 4][j % 4] = again[j];
      }
      __syncwarp();
    }
    if (GATED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[0][e] = n + e < p.n ? gate_f(sum[0][e], sum[TILES - 1][e], p.gate) : 0.f;
    }
    if (GATED && p.mode == OUT_FP8) {
      const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, max(max(fp8_abs_bits(sum[0][0]), fp8_abs_bits(sum[0][1])),
                                                                              max(fp8_abs_bits(sum[0][2]), fp8_abs_bits(sum[0][3])))));
      const uint32_t packed = fp8_pack4(sum[0][0], sum[0][1], sum[0][2], sum[0][3], fp8_inverse_scale(byte), byte);
      uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + (size_t)m * p.ldo + n;
      if (lane == 0) p.out_scales[(size_t)m * p.ldo_s + tile] = (uint8_t)byte;
      if (n + 4 <= p.n) {
        *reinterpret_cast<uint32_t*>(dst) = packed;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.n) dst[e] = (uint8_t)(packed >> (8 * e));
      }
    } else if (GATED || p.mode == OUT_BF16) {
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + (size_t)m * p.ldo + n;
      if (n + 4 <= p.n && p.vec_out) {
        uint2 pk;
        reinterpret_cast<__nv_bfloat162*>(&pk)[0] = __floats2bfloat162_rn(sum[0][0], sum[0][1]);
        reinterpret_cast<__nv_bfloat162*>(&pk)[1] = __floats2bfloat162_rn(sum[0][2], sum[0][3]);
        *reinterpret_cast<uint2*>(dst) = pk;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.n) dst[e] = __float2bfloat16_rn(sum[0][e]);
      }
    } else if (p.mode != OUT_ADD || nan == FAR_SUMS) {      // (nothing is added twice)
      float* dst = reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) sum[0][e] += p.mode == OUT_ADD ? dst[e] : 0.f;
      if (n + 4 <= p.n && p.vec_out) {
        *reinterpret_cast<float4*>(dst) = make_float4(sum[0][0], sum[0][1], sum[0][2], sum[0][3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.n) dst[e] = sum[0][e];
      }
    }
    if (GATED) nan = isnan((sum[0][0] + sum[0][1]) + (sum[0][2] + sum[0][3]));      // (of either side)
    return nan;
  };
  bool met = false;
  for (int i = here ? warp : own_tokens; i < own_tokens; i += WARPS) met = leave(i, std::false_type()) || met;
  // Everybody has sent (whoever has its sums knows that already).  A CTA that gave up waiting for them stays until they have landed.
  if (SLICED) {
    cluster_wait();
    if (!here) mbar_drain(sums_bar, 1, 1);
  }
  // (Last of all, so that the others end without a jump over it: 64 x 5,632 x 2,048 gated 10.8 us where it stood before the cluster's barrier.)
  if (!__any_sync(0xffffffffu, met)) return;
  for (int i = warp; i < own_tokens; i += WARPS) leave(i, std::true_type());
}

// ---------------------------------------------------------------- host side
// A 2-D tensor of bytes [rows, k] with row stride ld, tiled in boxes of box_rows x 128.
static bool make_map(CUtensorMap* map, const void* ptr, int rows, int k, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int STAGES, bool GATED>
static int launch_tiles(const Fp8Args& p, const void* a, long long lda, const void* w, long long ldw, int w_rows, int k, int* status, cudaStream_t s) {
  using L = Smem<BN, STAGES>;
  auto kern = linear_fp8_kernel<BN, STAGES, GATED>;
  TLLM_RESERVE_SMEM("linear_fp8", L::TOTAL, kern);
  CUtensorMap ma, mw;
  if (!make_map(&ma, a, p.m, k, lda, BM) || !make_map(&mw, w, w_rows, k, ldw, BN)) TLLM_FAIL(TLLM_ERR_CUDA, "linear_fp8: cannot describe the operands to the copy unit");
  // the registers that the summing warpgroups ask for are those of the launch, or they would wait for good
  static std::atomic<int> held{0};
  int regs = held.load(std::memory_order_relaxed);
  if (regs == 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess) TLLM_FAIL(TLLM_ERR_CUDA, "linear_fp8: cannot read the kernel's registers");
    held.store(regs = fa.numRegs, std::memory_order_relaxed);
  }
  TLLM_REQUIRE(regs * THREADS >= 32 * FIRST_SUM_WARP * REGS_OTHERS + 32 * SUM_WARPS * REGS_SUMS, "linear_fp8: built with %d registers, too few for its split", regs);
  const int tiles = ((p.m + BM - 1) / BM) * (GATED ? (p.n + 127) / 128 : (p.n + BN - 1) / BN);
  int dev = 0, sm_count = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sm_count < 1)
    TLLM_FAIL(TLLM_ERR_CUDA, "linear_fp8: cannot read the number of SMs");
  TLLM_LAUNCH("linear_fp8", kern, tiles < sm_count ? tiles : sm_count, THREADS, L::TOTAL, s, ma, mw, p, status);
  return TLLM_OK;
}

template <int BN, int STAGES, bool GATED, int HALVES, bool SLICED, int SENT = BN + 8>
static int launch_few(const Fp8Args& p, const FewArgs& f, const void* a, long long lda, const void* w, long long ldw, int w_rows, int k, int* status, cudaStream_t s) {
  using L = FewSmem<BN, STAGES, GATED, HALVES, SLICED, SENT>;
  auto kern = linear_fp8_few_kernel<BN, STAGES, GATED, HALVES, SLICED, SENT>;
  TLLM_RESERVE_SMEM("linear_fp8", L::TOTAL, kern);
  CUtensorMap ma, mw;
  if (!make_map(&mw, w, w_rows, k, ldw, 128) || !make_map(&ma, a, p.m, k, lda, BN)) TLLM_FAIL(TLLM_ERR_CUDA, "linear_fp8: cannot describe the operands to the copy unit");
  const int tiles = (p.n + 127) / 128, row_tiles = (p.m + BN - 1) / BN;
  TLLM_REQUIRE(tiles <= 65535, "linear_fp8: %d columns are too many for one launch", p.n);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_tiles, tiles, f.slices);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = f.slices;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mw, ma, p, f, status);
  if (e != cudaSuccess) TLLM_FAIL(TLLM_ERR_CUDA, "linear_fp8: %s", cudaGetErrorString(e));
  return TLLM_OK;
}

// How many clusters of `slices` CTAs the current device runs side by side: a cluster stays within a group of SMs, so that sizes that do
// not divide the group leave some of its SMs idle.  `alone`: with a CTA per SM (74 of two, 45 of three, 33, 26, 22, 15, 15; what the runtime
// answers for kernels that use tensor memory, however many of them fit an SM); `all`: with the RESIDENT ones that do run (two: 148, 93, 71, 56,
// 45, 37, 33; 296 CTAs of 128 values of K take 3.0 us, 297 4.4), which the runtime is asked about a kernel of the same size that does not.
// Asked once per kernel, size and device.
struct Clusters { int alone, all; };
template <int THREADS, int RESIDENT>
__global__ void __launch_bounds__(THREADS, RESIDENT) places_kernel() {}      // (never launched)
template <int BN, int STAGES, bool GATED, int HALVES, int SENT>
static Clusters most_clusters(int slices) {
  using L = FewSmem<BN, STAGES, GATED, HALVES, true, SENT>;
  static std::atomic<int> held[PerDeviceLimit::DEVICES][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= PerDeviceLimit::DEVICES) return {0, 0};
  const int known = held[dev][slices].load(std::memory_order_relaxed);
  if (known > 0) return {known >> 16, (known & 0xFFFF) - 1};
  auto kern = linear_fp8_few_kernel<BN, STAGES, GATED, HALVES, true, SENT>;
  auto places = places_kernel<L::THREADS, L::RESIDENT>;
  static PerDeviceLimit limit, places_limit;
  if (reserve_smem(limit, L::TOTAL, kern) != cudaSuccess || reserve_smem(places_limit, L::TOTAL, places) != cudaSuccess) return {0, 0};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, slices);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::TOTAL;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = slices;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  Clusters n = {};
  if (cudaOccupancyMaxActiveClusters(&n.alone, kern, &cfg) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n.all, places, &cfg) != cudaSuccess) return {0, 0};
  held[dev][slices].store((n.alone << 16) + n.all + 1, std::memory_order_relaxed);
  return n;
}

// Slices of K: as many as leave four groups to each, eight at most, and let all tiles run at once (6,144 x 4,096, 48 tiles: 6 slices in
// two rounds 9.5 us, 5 in one 6.6; 2,560 x 2,048: 8 slices of two groups 4.0, 4 of four 3.8).  Places where a cluster of one SM group's
// last CTAs shares SMs with its others are counted where the slices have twelve groups or more (8 rows, us without / with them: 4,096 columns, 32
// tiles on 33 places instead of 30, 8 slices of 4 groups 4.7 / 4.9, of 8 7.6 / 7.0, of 12 10.7 / 9.4, of 20 15.1 / 13.6; 8,960 columns, 70 on
// 71 instead of 66, 4 slices of 4 4.9 / 5.1, of 8 8.0 / 7.4, of 12 11.0 / 9.8; 7,040, 55 on 56 instead of 52, 5 slices of 8 7.7 / 8.1, of
// 12 10.4 / 10.6, of 64 rows 13.7 / 12.8).  Beyond them a second round begins (5,888, 46 on 45, 6 slices of 12: 10.4 / 14.8).
template <int BN, int STAGES, bool GATED, int HALVES, int SENT>
static int pick_slices(const Fp8Args& p) {
  const long long tiles = ((p.n + 127) / 128) * (long long)((p.m + BN - 1) / BN);
  for (int slices = min(8, p.groups / 4); slices > 1; --slices) {
    const Clusters most = most_clusters<BN, STAGES, GATED, HALVES, SENT>(slices);
    if (tiles <= (p.groups >= 12 * slices ? most.all : most.alone * FewSmem<BN, STAGES, GATED, HALVES, true, SENT>::RESIDENT)) return slices;
  }
  return 1;
}
template <int BN, int STAGES, int STAGES_WHOLE, bool GATED, int HALVES>     // (stages with slices, and without)
static int launch_few_rows(const Fp8Args& p, const void* a, long long lda, const void* w, long long ldw, int w_rows, int k, int* status, cudaStream_t s) {
  FewArgs f;
  f.slices = pick_slices<BN, STAGES, GATED, HALVES, BN + 8>(p);
  if (f.slices == 1) {
    f.per_slice = p.groups;
    return launch_few<BN, STAGES_WHOLE, GATED, HALVES, false, BN + 8>(p, f, a, lda, w, ldw, w_rows, k, status, s);
  }
  f.per_slice = (p.groups + f.slices - 1) / f.slices;
  f.slices = (p.groups + f.per_slice - 1) / f.per_slice;
  // Gated rows of a few tokens: the place for the sums is small enough for a third stage beside it, 96 KB of weights in flight per CTA
  // instead of 64 (8 rows of 5,632 x 2,048 7.2 us -> 5.8, of 2,816 x 2,048 6.0 -> 5.3).
  if constexpr (GATED && BN == 16) {
    if ((p.m + f.slices - 1) / f.slices * f.slices <= 9) return launch_few<BN, STAGES + 1, GATED, HALVES, true, 9>(p, f, a, lda, w, ldw, w_rows, k, status, s);
  }
  return launch_few<BN, STAGES, GATED, HALVES, true, BN + 8>(p, f, a, lda, w, ldw, w_rows, k, status, s);
}

// Few rows of A, or so few tiles that K has to be cut to fill the SMs: the weight's 128 rows as the large side (few), with as many rows
// of A beside them as keep what the CTAs fetch of the weight within 36 MB and them at once on the SMs (16 rows: one per SM): small tiles have the shorter
// way from the first product to the last store.  Otherwise tiles of 128 x 256 when they fill half the SMs, else of 128 x 128.
// us, few with 16 / 32 / 64 / 128 rows (columns x values of K):
//   2,560 x 2,048 of 32 rows 3.8 / 4.7 / 5.6 / 5.8, 64 4.8 / 5.0 / 6.2 / 5.8, 128 6.5 / 6.0 / 6.8 / 6.7, 256 12.2 / 8.6 / 8.6 / 8.4
//   4,096 x 4,096 of 64 7.8 / 7.1 / 8.3 / 8.2; 4,096 x 14,336 of 64 18.8 / 15.3 / 13.8 / 16.6
//   300 x 300 of 300 3.0 / 3.7 / 4.3 / 6.1; 1,000 x 1,520 of 333 6.3 / 5.8 / 7.1 / 6.7; 1,000 x 1,000 of 1,000 12.1 / 6.8 / 8.0 / 7.8
//   gated 5,632 x 2,048 of 32 8.4 / 8.1 / 9.1, 64 11.2 / 10.6 / 10.2; 300 x 300 of 300 4.5 / 5.4 / 6.8
// few / 128 x 128 / 128 x 256:
//   2,560 x 2,048 of 128 rows 7.1 / 9.6 / 13.4, 256 8.9 / 9.4 / 13.4, 512 11.2 / 9.8 / 13.7, 1,024 25 / 17.4 / 14.3
//   4,096 x 4,096 of 256 13.4 / 14.7 / 20, 512 20 / 14.8 / 20, 1,024 40 / 27 / 21
//   4,096 x 14,336 of 128 18.7 / 40 / 53, 256 32 / 40 / 53, 512 58 / 40 / 53, 1,024 116 / 78 / 59
// gated, few / 128 x 256: 5,632 x 2,048 of 64 rows 10.7 / 14.9, 128 14.2 / 15.4, 256 29 / 16; 14,336 x 4,096 of 64 23.7 / 26.4, 128 45 / 28
// (The columns' blocks are the second side of few's grid, which holds 65,535.)
// (Few: the rows of A per tile; tiles: 1,000 and their columns.)
enum Kernel { FEW_16 = 16, FEW_32 = 32, FEW_64 = 64, FEW_128 = 128, TILES_128 = 1128, TILES_256 = 1256 };
static Kernel pick_kernel(const Fp8Args& p, bool gated) {
  const long long m = p.m, w_tiles = (p.n + 127) / 128, w_values = (long long)p.w_rows * p.k;
  auto fits = [m, w_tiles, w_values](int rows, int resident) {
    const long long parts = (m + rows - 1) / rows;
    return w_tiles <= 65535 && (m <= rows || (parts * w_values <= 36000000 && parts * w_tiles <= 148 * resident));
  };
  const bool some = m <= 64 && w_tiles <= 65535;
  if (fits(16, 1)) return FEW_16;
  if (fits(32, gated ? 1 : 2)) return FEW_32;
  if (gated) return some || (m + 63) / 64 * w_tiles <= 148 ? FEW_64 : TILES_256;
  if (some) return FEW_64;
  if ((m + 127) / 128 * w_tiles <= 74) return FEW_128;
  return (m + 127) / 128 * ((p.n + 255) / 256) >= 74 ? TILES_256 : TILES_128;
}

}  // namespace tllm

using namespace tllm;

extern "C" const char* tllm_linear_fp8_layout() { return TLLM_LINEAR_FP8(TLLM_LETTER); }
// gated: `n` is the number of output columns, w has 256 * ceil(n / 128) rows; else w has n rows.
extern "C" int tllm_linear_fp8(const LinearFp8Call* c) {
  const auto [a, lda, a_scales, lda_s, w, ldw, w_scales, out, ldo, out_scales, ldo_s, m, n, k, mode, gated, act, limit, status_word, stream] = *c;
  int* status = (int*)status_word;
  TLLM_REQUIRE(m > 0 && n > 0 && k > 0, "linear_fp8: empty product");
  TLLM_REQUIRE(m <= FP8_MOST && n <= (gated ? FP8_MOST / 2 : FP8_MOST) && k <= FP8_MOST, "linear_fp8: at most %d rows of either operand and values per row", FP8_MOST);
  TLLM_REQUIRE((uintptr_t)a % 16 == 0 && (uintptr_t)w % 16 == 0 && lda % 16 == 0 && ldw % 16 == 0 && lda >= k && ldw >= k,
               "linear_fp8: rows of 8-bit values start on 16 bytes");
  TLLM_REQUIRE(gated ? (mode == OUT_BF16 || mode == OUT_FP8) : (mode >= OUT_BF16 && mode <= OUT_ADD), "linear_fp8: output code %d", mode);
  TLLM_REQUIRE(act >= 0 && act <= 3 && (act != ACT_CLAMPED || limit > 0.f), "linear_fp8: activation code %d, limit %g", act, (double)limit);
  Fp8Args p = {};
  p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.lda = lda; p.ldw = ldw; p.k = k;
  p.a_scales = (const uint8_t*)a_scales; p.w_scales = (const float*)w_scales; p.out = out; p.out_scales = (uint8_t*)out_scales;
  p.lda_s = lda_s; p.ldo = ldo; p.ldo_s = ldo_s;
  p.m = m; p.n = n; p.groups = (k + BK - 1) / BK;
  p.mode = mode; p.gate = make_gate(act, limit);
  const int size = mode == OUT_BF16 ? 2 : (mode == OUT_FP8 ? 1 : 4);
  p.vec_out = (uintptr_t)out % 16 == 0 && (ldo * size) % 16 == 0;
  p.vec_scales = (uintptr_t)a_scales % 4 == 0 && lda_s % 4 == 0;
  TLLM_REQUIRE(mode != OUT_FP8 || p.vec_out, "linear_fp8: rows of 8-bit values start on 16 bytes");
  cudaStream_t s = (cudaStream_t)stream;
  const int w_rows = gated ? 256 * ((n + 127) / 128) : n;
  p.w_rows = w_rows;
#define TLLM_FEW(BN, STAGES, WHOLE, GATED, HALVES) return launch_few_rows<BN, STAGES, WHOLE, GATED, HALVES>(p, a, lda, w, ldw, w_rows, k, status, s)
#define TLLM_TILES(BN, STAGES, GATED) return launch_tiles<BN, STAGES, GATED>(p, a, lda, w, ldw, w_rows, k, status, s)
  switch (pick_kernel(p, gated)) {
    case FEW_16: if (gated) TLLM_FEW(16, 2, 3, true, 1); else TLLM_FEW(16, 5, 6, false, 1);
    case FEW_32: if (gated) TLLM_FEW(32, 4, 5, true, 1); else TLLM_FEW(32, 4, 5, false, 1);
    case FEW_64: if (gated) TLLM_FEW(64, 3, 5, true, 2); else TLLM_FEW(64, 3, 4, false, 2);
    case FEW_128: TLLM_FEW(128, 4, 6, false, 4);
    case TILES_128: TLLM_TILES(128, 6, false);
    case TILES_256: if (gated) TLLM_TILES(256, 4, true); else TLLM_TILES(256, 4, false);
  }
#undef TLLM_FEW
#undef TLLM_TILES
  return TLLM_ERR_ARG;
}
// Which kernel a product of these sizes runs on, as Kernel numbers them, and into how many slices it cuts K on the current device: what the tests
// that name a kernel ask.
extern "C" int tllm_linear_fp8_kernel(int m, int n, int k, int gated, int* slices) {
  Fp8Args p = {};
  p.m = m; p.n = n; p.k = k; p.w_rows = gated ? 256 * ((n + 127) / 128) : n; p.groups = (k + BK - 1) / BK;
  const Kernel kernel = pick_kernel(p, gated);
  *slices = kernel == FEW_16 ? (gated ? pick_slices<16, 2, true, 1, 24>(p) : pick_slices<16, 5, false, 1, 24>(p))
          : kernel == FEW_32 ? (gated ? pick_slices<32, 4, true, 1, 40>(p) : pick_slices<32, 4, false, 1, 40>(p))
          : kernel == FEW_64 ? (gated ? pick_slices<64, 3, true, 2, 72>(p) : pick_slices<64, 3, false, 2, 72>(p))
          : kernel == FEW_128 ? pick_slices<128, 4, false, 4, 136>(p) : 1;
  return kernel;
}

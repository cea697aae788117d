// Rows and weights to 8 bits (e4m3) with a scale per group: see fp8.cuh for the rule.
//
//   * rows [M, K] of bfloat16 or float32: one scale (e8m0) per row and group of 128 values of K;
//   * the same behind a root-mean-square norm of float32 rows, so that the normed row never goes to memory;
//   * weights [N, K]: one float32 scale per block of 128 x 128.
// All are bound by memory: every value is read once (the norm's rows a second time where they do not fit the registers) and
// leaves as one byte.
#include <climits>
#include <type_traits>

#include "fp8.cuh"
#include "fp8_calls.h"

TLLM_DEFINE_LAST_ERROR

namespace tllm {

// four values from `src` + k on, zeros behind the last of `width`; `vec`: rows start where the wide load wants them
__device__ __forceinline__ void load4(const float* src, int k, int width, bool vec, float* v) {
  if (vec && k + 4 <= width) {
    const float4 f = *reinterpret_cast<const float4*>(src + k);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < width ? src[k + e] : 0.f;
  }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* src, int k, int width, bool vec, float* v) {
  if (vec && k + 4 <= width) {
    const uint2 u = *reinterpret_cast<const uint2*>(src + k);
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < width ? __bfloat162float(src[k + e]) : 0.f;
  }
}
// four bytes to `dst` + k (4-byte aligned), those before `width` only
__device__ __forceinline__ void store4(uint8_t* dst, int k, int width, uint32_t packed) {
  if (k + 4 <= width) {
    *reinterpret_cast<uint32_t*>(dst + k) = packed;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + e < width) dst[k + e] = (uint8_t)(packed >> (8 * e));
  }
}
__device__ __forceinline__ uint32_t largest4(const float* v) {
  return max(max(fp8_abs_bits(v[0]), fp8_abs_bits(v[1])), max(fp8_abs_bits(v[2]), fp8_abs_bits(v[3])));
}
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b) { a = __uint_as_float(u << 16); b = __uint_as_float(u & 0xFFFF0000u); }

// A warp's group of 128, four values per lane, to `dst` + k; returns the scale's byte.
__device__ __forceinline__ uint32_t leave_group(const float* v, uint8_t* dst, int k, int width) {
  const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, largest4(v)));
  store4(dst, k, width, fp8_pack4(v[0], v[1], v[2], v[3], fp8_inverse_scale(byte), byte));
  return byte;
}

constexpr int ROWS_THREADS = 256;

// A warp per row and run of groups, all of the run's loads in flight together: four groups of float32, four values per lane, or
// eight of bfloat16, eight values per lane and half a warp per group.  With 16-byte loads and no checks inside a run the kernel
// issues 25 instructions per group of bfloat16 instead of 86 and is bound by memory.
// Few groups: runs a quarter as long, so that four times the warps share the work.  us, long / short, by groups in all:
//   bfloat16  4,700 1.7 / 1.4 and 4.4 / 2.6 (rows of 2,048 and 1,000), 11,000 3.4 / 2.3, 16,500 3.8 / 2.3, 18,944 2.2 / 2.4, 22,000 3.7 / 2.6, 30,000 3.9 / 3.3,
//             40,000 4.0 / 4.0
//   float32   4,700 2.9 / 1.8, 9,500 2.0 / 2.3 and 2.4 / 2.2, 11,000 2.8 / 2.4, 12,500 2.7 / 2.6, 14,200 2.1 / 2.8, 16,500 2.9 / 3.1, 22,000 3.0 / 3.9
template <typename T> struct Run { static constexpr int LONG = 4, SHORT = 1, FEW = 148 * 84; };
template <> struct Run<__nv_bfloat16> { static constexpr int LONG = 8, SHORT = 2, FEW = 148 * 200; };

template <typename T, int GROUPS>
__global__ void __launch_bounds__(ROWS_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ out, long long ldo,
                     uint8_t* __restrict__ scales, long long lds, int rows, int width, int groups, int runs, int vec) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * (ROWS_THREADS / 32) + (threadIdx.x >> 5);
  const unsigned row = item / (unsigned)runs;
  if (row >= (unsigned)rows) return;
  const int g0 = (int)(item - row * runs) * GROUPS;
  const T* src = x + row * ldx;
  uint8_t* dst = out + row * ldo;
  uint32_t mine = 0u;      // lane i keeps the byte of the run's group i
  if (vec && (g0 + GROUPS) * FP8_GROUP <= width) {
    if constexpr (sizeof(T) == 2) {
      uint4 u[GROUPS / 2];
#pragma unroll
      for (int i = 0; i < GROUPS / 2; ++i) u[i] = *reinterpret_cast<const uint4*>(src + (g0 + 2 * i) * FP8_GROUP + 8 * lane);
#pragma unroll
      for (int i = 0; i < GROUPS / 2; ++i) {
        // magnitudes of bfloat16 are ordered as 16-bit integers, two to a word
        uint32_t most = __vmaxu2(__vmaxu2(u[i].x & 0x7FFF7FFFu, u[i].y & 0x7FFF7FFFu), __vmaxu2(u[i].z & 0x7FFF7FFFu, u[i].w & 0x7FFF7FFFu));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
        const uint32_t byte = fp8_scale_byte(max(most << 16, most & 0xFFFF0000u));
        const float inverse = fp8_inverse_scale(byte);
        float v[8];
        unpack2(u[i].x, v[0], v[1]); unpack2(u[i].y, v[2], v[3]); unpack2(u[i].z, v[4], v[5]); unpack2(u[i].w, v[6], v[7]);
        *reinterpret_cast<uint2*>(dst + (g0 + 2 * i) * FP8_GROUP + 8 * lane) =
            make_uint2(fp8_pack4(v[0], v[1], v[2], v[3], inverse, byte), fp8_pack4(v[4], v[5], v[6], v[7], inverse, byte));
        const uint32_t first = __shfl_sync(0xffffffffu, byte, 0), second = __shfl_sync(0xffffffffu, byte, 16);
        mine = lane == 2 * i ? first : lane == 2 * i + 1 ? second : mine;
      }
    } else {
      float4 f[GROUPS];
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) f[i] = *reinterpret_cast<const float4*>(src + (g0 + i) * FP8_GROUP + 4 * lane);
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const float v[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
        const uint32_t byte = leave_group(v, dst, (g0 + i) * FP8_GROUP + 4 * lane, width);
        mine = lane == i ? byte : mine;
      }
    }
  } else {
    constexpr int HALF = GROUPS < 4 ? GROUPS : 4;
    const bool vec4 = (reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int h = 0; h < GROUPS; h += HALF) {
      float v[HALF][4];
#pragma unroll
      for (int i = 0; i < HALF; ++i) load4(src, (g0 + h + i) * FP8_GROUP + 4 * lane, width, vec4, v[i]);   // (zeros behind the row's end)
#pragma unroll
      for (int i = 0; i < HALF; ++i) {
        if (g0 + h + i >= groups) break;
        const uint32_t byte = leave_group(v[i], dst, (g0 + h + i) * FP8_GROUP + 4 * lane, width);
        mine = lane == h + i ? byte : mine;
      }
    }
  }
  if (lane < GROUPS && g0 + lane < groups) scales[row * lds + g0 + lane] = (uint8_t)mine;
}

// A CTA per row: y = (w x) / sqrt(mean(x^2) + eps) in 32 bits.  A warp takes PER neighbouring groups, which stay in registers between
// the sum and the rounding, and stores their scales at once (PER = 0: every group that is left, read twice).  FULL: the row is whole groups, on 16 bytes.
template <int PER, bool FULL>
__device__ __forceinline__ void rms_norm_row(const float* __restrict__ x, const float* __restrict__ w, uint8_t* __restrict__ out, long long ldo,
                                             uint8_t* __restrict__ scales, long long lds, const int* __restrict__ gather, int width, int groups,
                                             float eps, int vec) {
  __shared__ float part[32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float* src = x + (size_t)(gather ? gather[blockIdx.x] : (int)blockIdx.x) * width;
  uint8_t* dst = out + (size_t)blockIdx.x * ldo;
  auto load = [&](const float* from, int g, float* v) {
    if (FULL) {
      const float4 f = g < groups ? *reinterpret_cast<const float4*>(from + g * FP8_GROUP + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      load4(from, g * FP8_GROUP + 4 * lane, width, vec, v);
    }
  };
  // the gains come in batches, the first while the row's sum is under way
  constexpr int BATCH = PER >= 4 ? 4 : PER > 0 ? PER : 1;
  float v[PER > 0 ? PER : 1][4], gain[BATCH][4], sum = 0.f;
  const int g0 = warp * PER;
  if (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) load(src, g0 + i, v[i]);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) load(w, g0 + i, gain[i]);
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += v[i][0] * v[i][0] + v[i][1] * v[i][1] + v[i][2] * v[i][2] + v[i][3] * v[i][3];
  } else {
    for (int g = warp; g < groups; g += warps) {
      load(src, g, v[0]);
      sum += v[0][0] * v[0][0] + v[0][1] * v[0][1] + v[0][2] * v[0][2] + v[0][3] * v[0][3];
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = warp_sum(lane < warps ? part[lane] : 0.f);
  const float inv = 1.f / sqrtf(sum / (float)width + eps);
  auto leave = [&](int g, float* y, const float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (f[e] * y[e]) * inv;
    return leave_group(y, dst, g * FP8_GROUP + 4 * lane, FULL ? INT_MAX : width);
  };
  uint8_t* row_scales = scales + (size_t)blockIdx.x * lds;
  if (PER > 0) {
    uint32_t mine = 0u;      // lane i keeps the byte of the warp's group i
#pragma unroll
    for (int h = 0; h < PER; h += BATCH) {
      if (h > 0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) load(w, g0 + h + i, gain[i]);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (g0 + h + i < groups) {
          const uint32_t byte = leave(g0 + h + i, v[h + i], gain[i]);
          mine = lane == h + i ? byte : mine;
        }
    }
    if (lane < PER && g0 + lane < groups) row_scales[g0 + lane] = (uint8_t)mine;
  } else {
    for (int g = warp; g < groups; g += warps) {
      load(src, g, v[0]);
      load(w, g, gain[0]);
      const uint32_t byte = leave(g, v[0], gain[0]);
      if (lane == 0) row_scales[g] = (uint8_t)byte;
    }
  }
}
template <int PER, bool FULL>
__global__ void rms_norm_rows_kernel(const float* __restrict__ x, const float* __restrict__ w, uint8_t* __restrict__ out, long long ldo,
                                     uint8_t* __restrict__ scales, long long lds, const int* __restrict__ gather, int width, int groups,
                                     float eps, int vec) {
  rms_norm_row<PER, FULL>(x, w, out, ldo, scales, lds, gather, width, groups, eps, vec);
}
// Eight groups per warp want 68 registers (79 where the row is not FULL), of which 28 (25) warps fit an SM.  Rows of more than NORM_WARPS warps
// run within the 64 that 32 warps may have; for the others that bound changed the order of the loads (2,048 rows of 2,048: 4.9 us,
// 5.2 with it; of 14,336 30.4 and 31.5).
constexpr int NORM_WARPS = 24;
template <bool FULL>
__global__ void __launch_bounds__(1024)
rms_norm_wide_rows_kernel(const float* __restrict__ x, const float* __restrict__ w, uint8_t* __restrict__ out, long long ldo,
                          uint8_t* __restrict__ scales, long long lds, const int* __restrict__ gather, int width, int groups, float eps, int vec) {
  rms_norm_row<8, FULL>(x, w, out, ldo, scales, lds, gather, width, groups, eps, vec);
}

constexpr int WEIGHT_THREADS = 512;

// four values of a lane as they came
template <typename T> struct Held { float4 v; };
template <> struct Held<__nv_bfloat16> { uint2 v; };
__device__ __forceinline__ void give(const Held<float>& h, float* v) { v[0] = h.v.x; v[1] = h.v.y; v[2] = h.v.z; v[3] = h.v.w; }
__device__ __forceinline__ void give(const Held<__nv_bfloat16>& h, float* v) { unpack2(h.v.x, v[0], v[1]); unpack2(h.v.y, v[2], v[3]); }
__device__ __forceinline__ void take(Held<float>& h, const float* src, int k, int width, bool vec) {
  if (vec && k + 4 <= width) { h.v = *reinterpret_cast<const float4*>(src + k); return; }
  float v[4];
  load4(src, k, width, false, v);
  h.v = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void take(Held<__nv_bfloat16>& h, const __nv_bfloat16* src, int k, int width, bool vec) {
  if (vec && k + 4 <= width) { h.v = *reinterpret_cast<const uint2*>(src + k); return; }
  float v[4];
  load4(src, k, width, false, v);
  h.v = make_uint2((__float_as_uint(v[0]) >> 16) | __float_as_uint(v[1]), (__float_as_uint(v[2]) >> 16) | __float_as_uint(v[3]));
}

// A CTA per block of 128 x 128, which stays in registers (bfloat16 as it came) between the search for its largest magnitude and the
// rounding.  The products may begin to read a weight, through the copy unit, before their wait for earlier launches: this kernel never lets
// the next one start early, and its values are in memory, for the copy unit too, before it ends.
template <typename T>
__global__ void __launch_bounds__(WEIGHT_THREADS, 3)
quantize_weight_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ out, long long ldo, float* __restrict__ scales,
                       int rows, int width, int groups, int vec) {
  constexpr int WARPS = WEIGHT_THREADS / 32, PER = FP8_GROUP / WARPS;
  __shared__ uint32_t most[WARPS];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = blockIdx.x * FP8_GROUP + 4 * lane, n0 = blockIdx.y * FP8_GROUP + warp;
  Held<T> held[PER];
  const T* src = w + (long long)n0 * ldw;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (n0 + i * WARPS < rows) take(held[i], src + (long long)i * WARPS * ldw, k, width, vec);
    else held[i].v = {};
  }
  uint32_t largest = 0u;
  float v[4];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    give(held[i], v);
    largest = max(largest, largest4(v));
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (lane == 0) most[warp] = largest;
  __syncthreads();
  largest = __reduce_max_sync(0xffffffffu, most[lane % WARPS]);
  const uint32_t byte = fp8_scale_byte(largest);
  const float inverse = fp8_inverse_scale(byte);
  uint8_t* dst = out + (long long)n0 * ldo;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    give(held[i], v);
    if (n0 + i * WARPS < rows) store4(dst + (long long)i * WARPS * ldo, k, width, fp8_pack4(v[0], v[1], v[2], v[3], inverse, byte));
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * groups + blockIdx.x] = fp8_scale(byte);
  __syncthreads();
  if (threadIdx.x == 0) {      // (behind the barrier, so for all threads' values)
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
  }
}

static int check_rows(const char* name, int rows, int width, const void* out, long long ldo, long long lds) {
  TLLM_REQUIRE(rows > 0 && width > 0, "%s: empty input", name);
  TLLM_REQUIRE(rows <= FP8_MOST && width <= FP8_MOST, "%s: at most %d rows and values per row", name, FP8_MOST);
  TLLM_REQUIRE((uintptr_t)out % 16 == 0 && ldo % 16 == 0 && ldo >= width, "%s: rows of 8-bit values start on 16 bytes", name);
  TLLM_REQUIRE(lds >= (width + 127ll) / 128, "%s: a row of scales holds one per group of 128", name);
  return TLLM_OK;
}

}  // namespace tllm

using namespace tllm;

// Entry points take their arguments as one struct; ..._layout() says how the interpreter packs it.
extern "C" const char* tllm_quantize_fp8_layout() { return TLLM_QUANTIZE_FP8(TLLM_LETTER); }
extern "C" int tllm_quantize_fp8(const QuantizeCall* c) {
  const auto [x, ldx, out, ldo, scales, lds, rows, width, dtype, stream] = *c;
  if (int e = check_rows("quantize_fp8", rows, width, out, ldo, lds)) return e;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  const bool few = (long long)rows * groups <= (dtype == TLLM_F32 ? Run<float>::FEW : Run<__nv_bfloat16>::FEW);
  const int run = dtype == TLLM_F32 ? (few ? Run<float>::SHORT : Run<float>::LONG) : (few ? Run<__nv_bfloat16>::SHORT : Run<__nv_bfloat16>::LONG);
  const int runs = (groups + run - 1) / run;
  TLLM_REQUIRE((long long)rows * runs < (1ll << 31), "quantize_fp8: %d rows of %d values are too many for one launch", rows, width);
  const unsigned blocks = ((unsigned)rows * runs + ROWS_THREADS / 32 - 1) / (ROWS_THREADS / 32);
  const int vec = (uintptr_t)x % 16 == 0 && ldx % (dtype == TLLM_F32 ? 4 : 8) == 0;
  cudaStream_t s = (cudaStream_t)stream;
#define TLLM_ROWS(T, GROUPS)                                                                                                      \
  TLLM_LAUNCH("quantize_fp8", (quantize_rows_kernel<T, GROUPS>), blocks, ROWS_THREADS, 0, s, (const T*)x, ldx, (uint8_t*)out, ldo, \
              (uint8_t*)scales, lds, rows, width, groups, runs, vec)
  if (dtype == TLLM_F32) {
    if (few) TLLM_ROWS(float, Run<float>::SHORT);
    else TLLM_ROWS(float, Run<float>::LONG);
  } else {
    if (few) TLLM_ROWS(__nv_bfloat16, Run<__nv_bfloat16>::SHORT);
    else TLLM_ROWS(__nv_bfloat16, Run<__nv_bfloat16>::LONG);
  }
#undef TLLM_ROWS
  return TLLM_OK;
}

extern "C" const char* tllm_rms_norm_fp8_layout() { return TLLM_RMS_NORM_FP8(TLLM_LETTER); }
extern "C" int tllm_rms_norm_fp8(const RmsNormCall* c) {
  const auto [x, w, out, ldo, scales, lds, rows_idx, rows, width, eps, stream] = *c;
  if (int e = check_rows("rms_norm_fp8", rows, width, out, ldo, lds)) return e;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  const int vec = (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && width % 4 == 0;
  // Few groups in all leave SMs idle: a warp per group is the shortest way through a row, up to 16 groups; more of them per warp where the row has
  // more.  Many groups: eight per warp, so that more rows fit an SM.  us, eight / fewer, by rows x values (groups in all):
  //   592 x 1,000 (4,736) 3.0 / 2.0, 320 x 2,048 (5,120) 4.1 / 2.5, 444 x 4,096 (14,208) 4.5 / 2.9, 592 x 4,096 (18,944) 4.6 / 3.8, 296 x 8,192
  //   (18,944) 4.1 / 3.3, 1,184 x 2,048 (18,944) 4.5 / 4.5, 320 x 8,192 (20,480) 4.1 / 4.5, 812 x 4,096 (25,984) 4.6 / 4.9, 1,625 x 2,048 (26,000) 4.6 / 5.7
  const bool few = (long long)rows * groups <= 148 * 128;
  const int per = !few ? 8 : groups <= 16 ? 1 : groups <= 32 ? 2 : groups <= 64 ? 4 : 8;
  const int warps = min(32, max(1, (groups + per - 1) / per));
  const bool full = vec && width % FP8_GROUP == 0;
  auto pick = [&](auto whole) {
    constexpr bool F = decltype(whole)::value;
    return warps * per < groups ? rms_norm_rows_kernel<0, F> : per == 1 ? rms_norm_rows_kernel<1, F> : per == 2 ? rms_norm_rows_kernel<2, F>
           : per == 4 ? rms_norm_rows_kernel<4, F> : warps <= NORM_WARPS ? rms_norm_rows_kernel<8, F> : rms_norm_wide_rows_kernel<F>;
  };
  auto kern = full ? pick(std::true_type()) : pick(std::false_type());
  TLLM_LAUNCH("rms_norm_fp8", kern, rows, 32 * warps, 0, (cudaStream_t)stream, (const float*)x, (const float*)w, (uint8_t*)out, ldo, (uint8_t*)scales, lds,
              (const int*)rows_idx, width, groups, eps, vec);
  return TLLM_OK;
}

extern "C" const char* tllm_quantize_weight_fp8_layout() { return TLLM_QUANTIZE_WEIGHT_FP8(TLLM_LETTER); }
extern "C" int tllm_quantize_weight_fp8(const QuantizeWeightCall* c) {
  const auto [w, ldw, out, ldo, scales, rows, width, dtype, stream] = *c;
  if (int e = check_rows("quantize_weight_fp8", rows, width, out, ldo, (width + 127ll) / 128)) return e;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  const int bytes = dtype == TLLM_F32 ? 4 : 2;
  const int vec = (uintptr_t)w % (4 * bytes) == 0 && ldw % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  constexpr int MOST_ROWS = 65535 * FP8_GROUP;      // of a launch: the second side of its grid (working the third one in cost every launch 5 to 10 %)
  for (long long r = 0; r < rows; r += MOST_ROWS) {
    const int some = rows - r < MOST_ROWS ? (int)(rows - r) : MOST_ROWS;
    const dim3 grid(groups, (some + FP8_GROUP - 1) / FP8_GROUP);
    const uint8_t* from = (const uint8_t*)w + r * ldw * bytes;
    uint8_t* to = (uint8_t*)out + r * ldo;
    float* to_scales = (float*)scales + r / FP8_GROUP * groups;
    if (dtype == TLLM_F32)
      TLLM_LAUNCH("quantize_weight_fp8", quantize_weight_kernel<float>, grid, WEIGHT_THREADS, 0, s, (const float*)from, ldw, to, ldo, to_scales, some, width, groups, vec);
    else
      TLLM_LAUNCH("quantize_weight_fp8", quantize_weight_kernel<__nv_bfloat16>, grid, WEIGHT_THREADS, 0, s, (const __nv_bfloat16*)from, ldw, to, ldo, to_scales, some, width, groups, vec);
  }
  return TLLM_OK;
}

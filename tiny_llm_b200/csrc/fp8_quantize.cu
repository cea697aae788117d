// Rows and weights to 8 bits (e4m3) with a scale per group: see fp8.cuh for the rule.
//
//   * rows [M, K] of bfloat16 or float32: one scale (e8m0) per row and group of 128 values of K;
//   * the same behind a root-mean-square norm of float32 rows, so that the normed row never goes to memory;
//   * weights [N, K]: one float32 scale per block of 128 x 128.
// All are bound by memory: every value is read once (the norm's rows a second time where they do not fit the registers) and
// leaves as one byte.
#include "fp8.cuh"

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

constexpr int ROWS_THREADS = 256;

// A warp per row and run of four groups: four values per lane and group, the four loads in flight together.
constexpr int ROWS_RUN = 4;
template <typename T>
__global__ void __launch_bounds__(ROWS_THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ out, long long ldo,
                     uint8_t* __restrict__ scales, long long lds, int rows, int width, int groups, int runs, int vec) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * (ROWS_THREADS / 32) + (threadIdx.x >> 5);
  const unsigned row = item / (unsigned)runs;
  if (row >= (unsigned)rows) return;
  const int g0 = (int)(item - row * runs) * ROWS_RUN;
  const T* src = x + row * ldx;
  float v[ROWS_RUN][4];
#pragma unroll
  for (int i = 0; i < ROWS_RUN; ++i) load4(src, (g0 + i) * FP8_GROUP + 4 * lane, width, vec, v[i]);   // (zeros behind the row's end)
#pragma unroll
  for (int i = 0; i < ROWS_RUN; ++i) {
    const int g = g0 + i, k = g * FP8_GROUP + 4 * lane;
    if (g >= groups) break;
    const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, largest4(v[i])));
    store4(out + row * ldo, k, width, fp8_pack4(v[i][0], v[i][1], v[i][2], v[i][3], fp8_inverse_scale(byte)));
    if (lane == 0) scales[row * lds + g] = (uint8_t)byte;
  }
}

// A CTA per row: y = (w x) / sqrt(mean(x^2) + eps) in 32 bits.  Warp i of W takes the groups i, i + W, ...: PER of them, which stay
// in registers between the sum and the rounding (PER = 0: any number, read twice).
template <int PER>
__global__ void rms_norm_rows_kernel(const float* __restrict__ x, const float* __restrict__ w, uint8_t* __restrict__ out, long long ldo,
                                     uint8_t* __restrict__ scales, long long lds, const int* __restrict__ gather, int width, int groups,
                                     float eps, int vec) {
  __shared__ float part[32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float* src = x + (size_t)(gather ? gather[blockIdx.x] : (int)blockIdx.x) * width;
  uint8_t* dst = out + (size_t)blockIdx.x * ldo;
  float v[PER > 0 ? PER : 1][4], f[PER > 0 ? PER : 1][4];
  float sum = 0.f;
  if (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) load4(src, (warp + i * warps) * FP8_GROUP + 4 * lane, width, vec, v[i]);
#pragma unroll
    for (int i = 0; i < PER; ++i) load4(w, (warp + i * warps) * FP8_GROUP + 4 * lane, width, vec, f[i]);
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += v[i][0] * v[i][0] + v[i][1] * v[i][1] + v[i][2] * v[i][2] + v[i][3] * v[i][3];
  } else {
    for (int g = warp; g < groups; g += warps) {
      load4(src, g * FP8_GROUP + 4 * lane, width, vec, v[0]);
      sum += v[0][0] * v[0][0] + v[0][1] * v[0][1] + v[0][2] * v[0][2] + v[0][3] * v[0][3];
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = warp_sum(lane < warps ? part[lane] : 0.f);
  const float inv = 1.f / sqrtf(sum / (float)width + eps);
  auto leave = [&](int g, float* y, const float* gain) {
    const int k = g * FP8_GROUP + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (gain[e] * y[e]) * inv;
    const uint32_t byte = fp8_scale_byte(__reduce_max_sync(0xffffffffu, largest4(y)));
    store4(dst, k, width, fp8_pack4(y[0], y[1], y[2], y[3], fp8_inverse_scale(byte)));
    if (lane == 0) scales[(size_t)blockIdx.x * lds + g] = (uint8_t)byte;
  };
  if (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (warp + i * warps < groups) leave(warp + i * warps, v[i], f[i]);
  } else {
    for (int g = warp; g < groups; g += warps) {
      load4(src, g * FP8_GROUP + 4 * lane, width, vec, v[0]);
      load4(w, g * FP8_GROUP + 4 * lane, width, vec, f[0]);
      leave(g, v[0], f[0]);
    }
  }
}

constexpr int WEIGHT_THREADS = 512;

// A CTA per block of 128 x 128, which stays in registers between the search for its largest magnitude and the rounding.  The
// products may begin to read a weight while earlier launches still run, so this kernel never lets the next one start early.
template <typename T>
__global__ void __launch_bounds__(WEIGHT_THREADS)
quantize_weight_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ out, long long ldo, float* __restrict__ scales,
                       int rows, int width, int groups, int vec) {
  constexpr int WARPS = WEIGHT_THREADS / 32, PER = FP8_GROUP / WARPS;
  __shared__ uint32_t most[WARPS];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = blockIdx.x * FP8_GROUP + 4 * lane, n0 = blockIdx.y * FP8_GROUP;
  float v[PER][4];
  uint32_t largest = 0u;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int n = n0 + i * WARPS + warp;
    if (n < rows) load4(w + n * ldw, k, width, vec, v[i]);
    else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) largest = max(largest, largest4(v[i]));
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (lane == 0) most[warp] = largest;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) largest = max(largest, most[i]);
  const uint32_t byte = fp8_scale_byte(largest);
  const float inverse = fp8_inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int n = n0 + i * WARPS + warp;
    if (n < rows) store4(out + n * ldo, k, width, fp8_pack4(v[i][0], v[i][1], v[i][2], v[i][3], inverse));
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * groups + blockIdx.x] = fp8_scale(byte);
  __threadfence();
}

static int check_rows(const char* name, int rows, int width, const void* out, long long ldo, long long lds) {
  TLLM_REQUIRE(rows > 0 && width > 0, "%s: empty input", name);
  TLLM_REQUIRE((uintptr_t)out % 16 == 0 && ldo % 16 == 0 && ldo >= width, "%s: rows of 8-bit values start on 16 bytes", name);
  TLLM_REQUIRE(lds >= (width + FP8_GROUP - 1) / FP8_GROUP, "%s: a row of scales holds one per group of 128", name);
  return TLLM_OK;
}

}  // namespace tllm

using namespace tllm;

// Entry points take their arguments as one struct, which the caller packs in the order of the declaration.
struct QuantizeCall { const void* x; long long ldx; void* out; long long ldo; void* scales; long long lds; int rows, width, dtype; void* stream; };
extern "C" int tllm_quantize_fp8(const QuantizeCall* c) {
  const auto [x, ldx, out, ldo, scales, lds, rows, width, dtype, stream] = *c;
  if (int e = check_rows("quantize_fp8", rows, width, out, ldo, lds)) return e;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  const int runs = (groups + ROWS_RUN - 1) / ROWS_RUN;
  TLLM_REQUIRE((long long)rows * runs < (1ll << 31), "quantize_fp8: %d rows of %d values are too many for one launch", rows, width);
  const unsigned blocks = ((unsigned)rows * runs + ROWS_THREADS / 32 - 1) / (ROWS_THREADS / 32);
  const int bytes = dtype == TLLM_F32 ? 16 : 8;
  const int vec = (uintptr_t)x % bytes == 0 && ldx % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TLLM_F32)
    TLLM_LAUNCH("quantize_fp8", quantize_rows_kernel<float>, blocks, ROWS_THREADS, 0, s, (const float*)x, ldx, (uint8_t*)out, ldo, (uint8_t*)scales, lds, rows, width, groups, runs, vec);
  else
    TLLM_LAUNCH("quantize_fp8", quantize_rows_kernel<__nv_bfloat16>, blocks, ROWS_THREADS, 0, s, (const __nv_bfloat16*)x, ldx, (uint8_t*)out, ldo, (uint8_t*)scales, lds, rows, width, groups, runs, vec);
  return TLLM_OK;
}

struct RmsNormCall { const float *x, *w; void* out; long long ldo; void* scales; long long lds; const int* rows_idx; int rows, width; float eps; void* stream; };
extern "C" int tllm_rms_norm_fp8(const RmsNormCall* c) {
  const auto [x, w, out, ldo, scales, lds, rows_idx, rows, width, eps, stream] = *c;
  if (int e = check_rows("rms_norm_fp8", rows, width, out, ldo, lds)) return e;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  const int vec = (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && width % 4 == 0;
  // Few rows leave most SMs idle: a warp per group is the shortest way through a row.  Many rows: eight groups per warp, so that more
  // rows fit an SM.
  const int per = rows <= 296 ? (groups <= 16 ? 1 : groups <= 32 ? 2 : groups <= 64 ? 4 : 8) : 8;
  const int warps = min(32, max(1, (groups + per - 1) / per));
  auto kern = warps * per < groups ? rms_norm_rows_kernel<0> : per == 1 ? rms_norm_rows_kernel<1> : per == 2 ? rms_norm_rows_kernel<2>
              : per == 4 ? rms_norm_rows_kernel<4> : rms_norm_rows_kernel<8>;
  TLLM_LAUNCH("rms_norm_fp8", kern, rows, 32 * warps, 0, (cudaStream_t)stream, x, w, (uint8_t*)out, ldo, (uint8_t*)scales, lds, rows_idx, width, groups, eps, vec);
  return TLLM_OK;
}

struct QuantizeWeightCall { const void* w; long long ldw; void* out; long long ldo; float* scales; int rows, width, dtype; void* stream; };
extern "C" int tllm_quantize_weight_fp8(const QuantizeWeightCall* c) {
  const auto [w, ldw, out, ldo, scales, rows, width, dtype, stream] = *c;
  const int groups = (width + FP8_GROUP - 1) / FP8_GROUP;
  if (int e = check_rows("quantize_weight_fp8", rows, width, out, ldo, groups)) return e;
  const int row_blocks = (rows + FP8_GROUP - 1) / FP8_GROUP;
  TLLM_REQUIRE(row_blocks <= 65535, "quantize_weight_fp8: %d rows are too many for one launch", rows);
  const int bytes = dtype == TLLM_F32 ? 16 : 8;
  const int vec = (uintptr_t)w % bytes == 0 && ldw % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid(groups, row_blocks);
  if (dtype == TLLM_F32)
    TLLM_LAUNCH("quantize_weight_fp8", quantize_weight_kernel<float>, grid, WEIGHT_THREADS, 0, s, (const float*)w, ldw, (uint8_t*)out, ldo, scales, rows, width, groups, vec);
  else
    TLLM_LAUNCH("quantize_weight_fp8", quantize_weight_kernel<__nv_bfloat16>, grid, WEIGHT_THREADS, 0, s, (const __nv_bfloat16*)w, ldw, (uint8_t*)out, ldo, scales, rows, width, groups, vec);
  return TLLM_OK;
}

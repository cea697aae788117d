// The arguments of the 8-bit operators' entry points, as one struct each.  Every field is named once, here: the structs of the kernels' sources
// and of the calls' extension come from these lists, and so do the letters that the interpreter packs them by (P: pointer, q: 64 bits,
// i: 32 bits, f: float, in the machine's own alignment).  Plain C++, no CUDA.
#pragma once

#define TLLM_P void*
#define TLLM_q long long
#define TLLM_i int
#define TLLM_f float

#define TLLM_QUANTIZE_FP8(F) \
  F(P, x) F(q, ldx) F(P, out) F(q, ldo) F(P, scales) F(q, lds) F(i, rows) F(i, width) F(i, dtype) F(P, stream)
#define TLLM_RMS_NORM_FP8(F) \
  F(P, x) F(P, w) F(P, out) F(q, ldo) F(P, scales) F(q, lds) F(P, rows_idx) F(i, rows) F(i, width) F(f, eps) F(P, stream)
#define TLLM_QUANTIZE_WEIGHT_FP8(F) \
  F(P, w) F(q, ldw) F(P, out) F(q, ldo) F(P, scales) F(i, rows) F(i, width) F(i, dtype) F(P, stream)
#define TLLM_LINEAR_FP8(F) \
  F(P, a) F(q, lda) F(P, a_scales) F(q, lda_s) F(P, w) F(q, ldw) F(P, w_scales) F(P, out) F(q, ldo) F(P, out_scales) F(q, ldo_s) \
  F(i, m) F(i, n) F(i, k) F(i, mode) F(i, gated) F(i, act) F(f, limit) F(P, status) F(P, stream)

#define TLLM_FIELD(kind, name) TLLM_##kind name{};
#define TLLM_LETTER(kind, name) #kind
struct QuantizeCall { TLLM_QUANTIZE_FP8(TLLM_FIELD) };
struct RmsNormCall { TLLM_RMS_NORM_FP8(TLLM_FIELD) };
struct QuantizeWeightCall { TLLM_QUANTIZE_WEIGHT_FP8(TLLM_FIELD) };
struct LinearFp8Call { TLLM_LINEAR_FP8(TLLM_FIELD) };

// What the int8 product's kernels share: the outputs' scales and types.
#pragma once
#include "common.cuh"

namespace mtp {
namespace i8 {

constexpr int MAX_COLS = 131071;  // of a row: 128 * 128 * MAX_COLS < 2^31

struct Out {
  void *p;
  int64_t ld;
  int dtype;
  const float *a_scale, *w_scale;
  const void *bias;
  int bias_dtype;
};

__device__ __forceinline__ float ld_bias(const Out &o, int n) {
  if (!o.bias) return 0.f;
  if (o.bias_dtype == MTP_F32) return ((const float *)o.bias)[n];
  if (o.bias_dtype == MTP_BF16) return __bfloat162float(((const __nv_bfloat16 *)o.bias)[n]);
  return __half2float(((const __half *)o.bias)[n]);
}

// The result of a sum, in fp32 operations of a fixed order, so that every kernel gives the same bits.
__device__ __forceinline__ float scaled(int acc, float a_scale, float w_scale) {
  return __fmul_rn(__fmul_rn((float)acc, a_scale), w_scale);
}

__device__ __forceinline__ void store_value(const Out &o, int64_t m, int n, float v) {
  if (o.dtype == MTP_F32) ((float *)o.p)[m * o.ld + n] = v;
  else if (o.dtype == MTP_BF16) ((__nv_bfloat16 *)o.p)[m * o.ld + n] = __float2bfloat16_rn(v);
  else ((__half *)o.p)[m * o.ld + n] = __float2half_rn(v);
}

// Tensor-core form.  False from `eligible`: the operands are not on 16-byte boundaries.
bool tc_eligible(const int8_t *a, int64_t ld_a, int M, const int8_t *w, int64_t ld_w, int N);
int linear_tc(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o,
              cudaStream_t stream);

// For few tokens; operands on 16-byte boundaries as above.  (17 rows x 4096 -> 2048: 9.2 us here in three groups of 8, 6.7 in
// the tensor-core form; 16 rows 4.2.)
constexpr int FEW = 16;
int linear_few(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o,
               cudaStream_t stream);

}  // namespace i8
}  // namespace mtp

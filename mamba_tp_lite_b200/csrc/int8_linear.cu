// out[M, N] = (a[M, K] . w[N, K]^T) * a_scale[m] * w_scale[n] (+ bias): int8 operands, int32 sums.
//   int8_few.cu  up to 16 rows, operands on 16-byte boundaries;
//   int8_tc.cu   more rows, operands on 16-byte boundaries;
//   int8_simt    here: 64 x 64 tiles, 4 x 4 outputs per thread, byte loads: operands of any alignment (333 x 1001 -> 777 with
//                rows of 1001 bytes: 59 us; quantize_rows puts rows on 16-byte boundaries, 6.6 us).
#include "int8_linear.cuh"

namespace mtp {
namespace {

using namespace i8;

__global__ void __launch_bounds__(256) int8_simt_kernel(const int8_t *__restrict__ a, int64_t ld_a, int M, int K,
                                                        const int8_t *__restrict__ w, int64_t ld_w, int N, int tiles_n,
                                                        int64_t tiles, Out o) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ int as[16][65], ws[16][65];  // [4 values of k][row]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / tiles_n * 64;
    const int n0 = (int)(t % tiles_n) * 64;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 64) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int el = tid + i * 256, r = el >> 4, kk = el & 15;
        uint32_t va = 0, vw = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int k = k0 + 4 * kk + b;
          if (k < K && m0 + r < M) va |= (uint32_t)(uint8_t)a[(m0 + r) * ld_a + k] << (8 * b);
          if (k < K && n0 + r < N) vw |= (uint32_t)(uint8_t)w[(int64_t)(n0 + r) * ld_w + k] << (8 * b);
        }
        as[kk][r] = (int)va;
        ws[kk][r] = (int)vw;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < 16; ++kk) {
        int x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = as[kk][ty + 16 * i]; y[i] = ws[kk][tx + 16 * i]; }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + ty + 16 * i;
        const int n = n0 + tx + 16 * j;
        if (m < M && n < N) {
          float v = scaled(acc[i][j], o.a_scale[m], o.w_scale[n]);
          if (o.bias) v = __fadd_rn(v, ld_bias(o, n));
          store_value(o, m, n, v);
        }
      }
  }
}

bool dtype_ok(int d) { return d == MTP_F32 || d == MTP_BF16 || d == MTP_F16; }

}  // namespace
}  // namespace mtp

using namespace mtp;

extern "C" int mtp_int8_linear(const int8_t *a, int64_t ld_a, const float *a_scale, int M, int K, const int8_t *w,
                               int64_t ld_w, const float *w_scale, int N, const void *bias, int bias_dtype, void *out,
                               int out_dtype, int64_t ld_out, void *stream) {
  MTP_REQUIRE(M >= 0 && N >= 0 && K >= 1 && K <= MAX_COLS, "M and N must not be negative, K must be 1 to 131071");
  MTP_REQUIRE(dtype_ok(out_dtype) && (!bias || dtype_ok(bias_dtype)), "dtype must be F32, BF16 or F16");
  if (M == 0 || N == 0) return MTP_OK;
  MTP_REQUIRE(a && a_scale && w && w_scale && out, "null pointer");
  MTP_REQUIRE((M == 1 || (ld_a >= K && ld_out >= N)) && (N == 1 || ld_w >= K), "leading dimensions too small");
  cudaStream_t s = (cudaStream_t)stream;
  const Out o{out, ld_out, out_dtype, a_scale, w_scale, bias, bias_dtype};
  if (M <= FEW && tc_eligible(a, ld_a, M, w, ld_w, N)) return linear_few(a, ld_a, M, K, w, ld_w, N, o, s);
  if (tc_eligible(a, ld_a, M, w, ld_w, N)) return linear_tc(a, ld_a, M, K, w, ld_w, N, o, s);
  const int tiles_n = ceil_div(N, 64);
  const int64_t tiles = (int64_t)ceil_div(M, 64) * tiles_n;
  const int grid = (int)(tiles < 148 * 16 ? tiles : 148 * 16);
  launch_pdl(int8_simt_kernel, dim3(grid), dim3(256), 0, s, a, ld_a, M, K, w, ld_w, N, tiles_n, tiles, o);
  return check_launch("int8_linear");
}

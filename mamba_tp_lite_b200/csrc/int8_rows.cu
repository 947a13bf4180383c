// Rows of int8 codes with a scale each: quantising, reading back, and RMSNorm with the residual's addition and an int8
// output.  A CTA takes one row: a pass for its statistics, a pass for its codes.
#include "common.cuh"

namespace mtp {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_COLS = 131071;  // 127 * 127 * MAX_COLS < 2^31

__device__ __forceinline__ double block_reduce(double v, bool sum, double *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, o);
    v = sum ? v + u : fmax(v, u);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < THREADS / 32; ++i) v = sum ? v + red[i] : fmax(v, red[i]);
  return v;
}

// fp32 scale of a row whose largest |y| is amax; NaN for a row with a NaN or an infinity (`bad`).
__device__ __forceinline__ float scale_of(double amax, bool bad) {
  const float s = (float)(fmax(amax, 1e-8) / 127.0);
  return bad || !(s <= 3.402823466e38f) ? __int_as_float(0x7fffffff) : s;
}

__device__ __forceinline__ int8_t code_of(double y, float s) {
  return (int8_t)(int)fmin(fmax(rint(y / (double)s), -127.0), 127.0);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T *__restrict__ x, int64_t ld, int64_t rows, int cols,
                                                           int8_t *__restrict__ codes, int64_t ld_codes,
                                                           float *__restrict__ scale) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ double red[THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * ld;
    double amax = 0.0;
    bool bad = false;
    for (int c = threadIdx.x; c < cols; c += THREADS) {
      const float v = fabsf(ldf(xr + c));
      bad |= !(v <= 3.402823466e38f);
      amax = fmax(amax, (double)v);
    }
    amax = block_reduce(amax, false, red);
    bad = __syncthreads_or(bad);
    const float s = scale_of(amax, bad);
    for (int c = threadIdx.x; c < cols; c += THREADS)
      codes[r * ld_codes + c] = bad ? 0 : code_of((double)ldf(xr + c), s);
    if (threadIdx.x == 0) scale[r] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const int8_t *__restrict__ codes, int64_t ld_codes,
                                                             const float *__restrict__ scale, int64_t rows, int cols,
                                                             T *__restrict__ out, int64_t ld_out) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += THREADS)
      stf(out + r * ld_out + c, __fmul_rn((float)codes[r * ld_codes + c], scale[r]));
}

__device__ __forceinline__ float ld_any(const void *p, int dtype, int64_t i) {
  if (dtype == MTP_F32) return ((const float *)p)[i];
  if (dtype == MTP_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
  return __half2float(((const __half *)p)[i]);
}
__device__ __forceinline__ float st_any(void *p, int dtype, int64_t i, float v) {  // the value as it is held
  if (dtype == MTP_F32) return ((float *)p)[i] = v;
  if (dtype == MTP_BF16) {
    const __nv_bfloat16 h = __float2bfloat16_rn(v);
    ((__nv_bfloat16 *)p)[i] = h;
    return __bfloat162float(h);
  }
  const __half h = __float2half_rn(v);
  ((__half *)p)[i] = h;
  return __half2float(h);
}

__global__ void __launch_bounds__(THREADS)
    rmsnorm_int8_kernel(const void *x, int x_dtype, int64_t ld_x, const void *resid, int r_dtype, int64_t ld_r, void *r_out,
                        int64_t ld_ro, int64_t rows, int cols, const void *w, int w_dtype, float eps, int8_t *codes,
                        int64_t ld_codes, float *scale) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ double red[THREADS / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    double ss = 0.0;
    for (int c = threadIdx.x; c < cols; c += THREADS) {
      float h = ld_any(x, x_dtype, r * ld_x + c);
      if (resid) h = st_any(r_out, r_dtype, r * ld_ro + c, h + ld_any(resid, r_dtype, r * ld_r + c));
      ss += (double)h * (double)h;
    }
    ss = block_reduce(ss, true, red);
    const double rs = 1.0 / sqrt(ss / cols + (double)eps);
    // a thread reads back what it has stored itself
    const void *hp = resid ? r_out : x;
    const int h_dtype = resid ? r_dtype : x_dtype;
    const int64_t ld_h = resid ? ld_ro : ld_x;
    double amax = 0.0;
    bool bad = false;
    for (int c = threadIdx.x; c < cols; c += THREADS) {
      const double y = fabs((double)ld_any(hp, h_dtype, r * ld_h + c) * rs * (double)ld_any(w, w_dtype, c));
      bad |= !(y <= 1e300);
      amax = fmax(amax, y);
    }
    amax = block_reduce(amax, false, red);
    float s = scale_of(amax, __syncthreads_or(bad));
    bad = !(s > 0.f);
    for (int c = threadIdx.x; c < cols; c += THREADS) {
      const double y = (double)ld_any(hp, h_dtype, r * ld_h + c) * rs * (double)ld_any(w, w_dtype, c);
      codes[r * ld_codes + c] = bad ? 0 : code_of(y, s);
    }
    if (threadIdx.x == 0) scale[r] = s;
  }
}

int grid_for(int64_t rows) { return (int)(rows < 148 * 64 ? rows : 148 * 64); }

bool dtype_ok(int d) { return d == MTP_F32 || d == MTP_BF16 || d == MTP_F16; }
bool rows_ok(int64_t rows, int cols) { return rows >= 0 && rows <= 0x7fffffffll && cols >= 1 && cols <= MAX_COLS; }

}  // namespace
}  // namespace mtp

using namespace mtp;

#define MTP_DISPATCH_3(code, T, ...)                                        \
  do {                                                                      \
    if ((code) == MTP_F32) { using T = float; __VA_ARGS__; }                \
    else if ((code) == MTP_BF16) { using T = __nv_bfloat16; __VA_ARGS__; } \
    else { using T = __half; __VA_ARGS__; }                                 \
  } while (0)

extern "C" {

int mtp_quantize_rows(const void *x, int dtype, int64_t ld, int64_t rows, int cols, int8_t *codes, int64_t ld_codes,
                      float *scale, void *stream) {
  MTP_REQUIRE(rows_ok(rows, cols), "rows must be 0 to 2^31 - 1 and cols 1 to 131071");
  MTP_REQUIRE(dtype_ok(dtype), "dtype must be F32, BF16 or F16");
  if (rows == 0) return MTP_OK;
  MTP_REQUIRE(x && codes && scale, "null pointer");
  MTP_REQUIRE((rows == 1 || ld >= cols) && (rows == 1 || ld_codes >= cols), "leading dimensions too small");
  cudaStream_t s = (cudaStream_t)stream;
  MTP_DISPATCH_3(dtype, T, launch_pdl(quantize_kernel<T>, dim3(grid_for(rows)), dim3(THREADS), 0, s, (const T *)x, ld, rows,
                                      cols, codes, ld_codes, scale));
  return check_launch("quantize_rows");
}

int mtp_dequantize_rows(const int8_t *codes, int64_t ld_codes, const float *scale, int64_t rows, int cols, void *out,
                        int out_dtype, int64_t ld_out, void *stream) {
  MTP_REQUIRE(rows_ok(rows, cols), "rows must be 0 to 2^31 - 1 and cols 1 to 131071");
  MTP_REQUIRE(dtype_ok(out_dtype), "out_dtype must be F32, BF16 or F16");
  if (rows == 0) return MTP_OK;
  MTP_REQUIRE(codes && scale && out, "null pointer");
  MTP_REQUIRE(rows == 1 || (ld_codes >= cols && ld_out >= cols), "leading dimensions too small");
  cudaStream_t s = (cudaStream_t)stream;
  MTP_DISPATCH_3(out_dtype, T, launch_pdl(dequantize_kernel<T>, dim3(grid_for(rows)), dim3(THREADS), 0, s, codes, ld_codes,
                                          scale, rows, cols, (T *)out, ld_out));
  return check_launch("dequantize_rows");
}

int mtp_rmsnorm_int8(const void *x, int x_dtype, int64_t ld_x, const void *resid, int resid_dtype, int64_t ld_resid,
                     void *resid_out, int64_t ld_resid_out, int64_t rows, int cols, const void *w, int w_dtype,
                     float eps, int8_t *codes, int64_t ld_codes, float *scale, void *stream) {
  MTP_REQUIRE(rows_ok(rows, cols), "rows must be 0 to 2^31 - 1 and cols 1 to 131071");
  MTP_REQUIRE(dtype_ok(x_dtype) && dtype_ok(w_dtype) && (!resid || dtype_ok(resid_dtype)), "dtype must be F32, BF16 or F16");
  MTP_REQUIRE(eps >= 0.f, "eps must not be negative");
  if (rows == 0) return MTP_OK;
  MTP_REQUIRE(x && w && codes && scale && (!resid || resid_out), "null pointer");
  MTP_REQUIRE(rows == 1 || (ld_x >= cols && ld_codes >= cols && (!resid || (ld_resid >= cols && ld_resid_out >= cols))),
              "leading dimensions too small");
  cudaStream_t s = (cudaStream_t)stream;
  launch_pdl(rmsnorm_int8_kernel, dim3(grid_for(rows)), dim3(THREADS), 0, s, x, x_dtype, ld_x, resid, resid_dtype, ld_resid,
             resid_out, ld_resid_out, rows, cols, w, w_dtype, eps, codes, ld_codes, scale);
  return check_launch("rmsnorm_int8");
}

}  // extern "C"

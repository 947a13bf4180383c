// The int8 product for few tokens (a decode step): bound by reading w once.
//
// A CTA takes 16 channels and all of K: its warps split K into slices of 256 bytes, so that a warp's loads are all in flight
// together, and the slices' int32 sums are added in shared memory (exact in any order).  The products go through
// mma.m16n8k32: 16 channels by 8 tokens.  A lane's 16 bytes of a row are not those that the instruction's layout gives it, but
// it takes the same ones of w and of the tokens, and the order of k within a sum does not matter.
// Measured on a B200, L2 cold (us; w at 6550 GB/s): 1 x 2048 -> 8192 5.5 (2.6), 1 x 4096 -> 2048 3.5 (1.3), 16 rows 6.0 and
// 4.2, 1 x 2048 -> 50280 20.5 (15.7).  About 1 us is the launch, 1.5 the way of one load and of the sums through the CTA.
#include "int8_linear.cuh"

namespace mtp {
namespace i8 {
namespace {

constexpr int SLICE = 256, STEPS = SLICE / 64, MAX_WARPS = 16;

// 16 bytes of a row at k, those from K on zero.
__device__ __forceinline__ uint4 load_tail(const int8_t *row, int k, int K) {
  uint32_t w[4] = {};
  if (k + 16 <= K) return *reinterpret_cast<const uint4 *>(row + k);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void prefetch_line(const int8_t *p, bool on) {
  if (on) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

__device__ __forceinline__ void mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// PER_SM CTAs of 16 warps fit an SM.
template <int NT, int PER_SM>
__global__ void __launch_bounds__(32 * MAX_WARPS, PER_SM)
    int8_few_kernel(const int8_t *__restrict__ a, int64_t ld_a, int M, int K, const int8_t *__restrict__ w, int64_t ld_w, int N,
                    Out o) {
  __shared__ int sums[MAX_WARPS * NT * 8 * 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5;
  const int n0 = blockIdx.x * 16;
  // a lane whose channel or token does not exist takes the last one's: its sums are not used
  const int8_t *w0 = w + (int64_t)min(n0 + g, N - 1) * ld_w + 16 * t, *w1 = w + (int64_t)min(n0 + g + 8, N - 1) * ld_w + 16 * t;
  MTP_PDL_TRIGGER();
  if (t == 0) {  // w on its way to L2 (where a write of the kernel before would meet it) while that kernel ends
    for (int k = warp * SLICE; k < K; k += warps * SLICE) {
      prefetch_line(w0 + k, true);
      prefetch_line(w0 + k + 128, k + 128 < K);
      prefetch_line(w1 + k, true);
      prefetch_line(w1 + k + 128, k + 128 < K);
    }
  }
  MTP_PDL_WAIT();
  int acc[NT][4] = {};
  for (int k0 = warp * SLICE; k0 < K; k0 += warps * SLICE) {
    uint4 u[STEPS], v[STEPS];
    if (k0 + SLICE <= K) {
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        u[j] = __ldg(reinterpret_cast<const uint4 *>(w0 + k0 + 64 * j));
        v[j] = __ldg(reinterpret_cast<const uint4 *>(w1 + k0 + 64 * j));
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int8_t *row = a + (int64_t)min(8 * i + g, M - 1) * ld_a + 16 * t + k0;
        uint4 x[STEPS];
#pragma unroll
        for (int j = 0; j < STEPS; ++j) x[j] = __ldg(reinterpret_cast<const uint4 *>(row + 64 * j));
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          mma(acc[i], u[j].x, v[j].x, u[j].y, v[j].y, x[j].x, x[j].y);
          mma(acc[i], u[j].z, v[j].z, u[j].w, v[j].w, x[j].z, x[j].w);
        }
      }
    } else {
#pragma unroll 1
      for (int k = k0; k < K; k += 64) {
        const uint4 p = load_tail(w0, k, K - 16 * t), q = load_tail(w1, k, K - 16 * t);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint4 x = load_tail(a + (int64_t)min(8 * i + g, M - 1) * ld_a + 16 * t, k, K - 16 * t);
          mma(acc[i], p.x, q.x, p.y, q.y, x.x, x.y);
          mma(acc[i], p.z, q.z, p.w, q.w, x.z, x.w);
        }
      }
    }
  }
  // [warp][token][channel]
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    int *s = sums + ((warp * NT + i) * 8 + 2 * t) * 16 + g;
    s[0] = acc[i][0];
    s[16] = acc[i][1];
    s[8] = acc[i][2];
    s[24] = acc[i][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * M; e += blockDim.x) {
    const int n = n0 + (e & 15), m = e >> 4;
    int sum = 0;
    for (int i = 0; i < warps; ++i) sum += sums[i * NT * 128 + e];
    if (n < N) {
      float y = scaled(sum, o.a_scale[m], o.w_scale[n]);
      if (o.bias) y = __fadd_rn(y, ld_bias(o, n));
      store_value(o, m, n, y);
    }
  }
}

template <int NT>
void launch(dim3 grid, dim3 block, cudaStream_t s, const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w,
            int N, const Out &o) {
  // Two CTAs per SM where there are more than SMs (1 x 2048 -> 8192: 5.6 us, with one 6.2); with one CTA for each SM, room for
  // one only, since early launches of the next kernel would else crowd some SMs (1 x 4096 -> 2048: 3.5 us, with two 4.5).
  if ((int)grid.x <= num_sms()) launch_pdl(int8_few_kernel<NT, 1>, grid, block, 0, s, a, ld_a, M, K, w, ld_w, N, o);
  else launch_pdl(int8_few_kernel<NT, 2>, grid, block, 0, s, a, ld_a, M, K, w, ld_w, N, o);
}

}  // namespace

int linear_few(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o,
               cudaStream_t stream) {
  const int slices = ceil_div(K, SLICE);
  const dim3 grid(ceil_div(N, 16)), block(32 * (slices < MAX_WARPS ? slices : MAX_WARPS));
  if (M <= 8) launch<1>(grid, block, stream, a, ld_a, M, K, w, ld_w, N, o);
  else launch<2>(grid, block, stream, a, ld_a, M, K, w, ld_w, N, o);
  return check_launch("int8_linear");
}

}  // namespace i8
}  // namespace mtp

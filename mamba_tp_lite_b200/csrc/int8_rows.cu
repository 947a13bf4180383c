// Rows of int8 codes with a scale each: quantising, reading back, and RMSNorm with the residual's addition and an int8
// output.
//
// Bound by HBM, or for a row at a time by latency.  A row belongs to a team of threads (a warp, or a CTA) that keeps it in
// registers, so that it is read once; vectors of 16 bytes, shifted together from two where rows do not lie on such boundaries.
// Which of two codes is the nearer is decided as in exact arithmetic without 64 bits for each value: a value held exactly leaves
// an exact remainder in fp32 (exact_codes4); a norm's quotient is known to 3e-5 of a step in fp32, and only where it is within
// 2^-14 of a half (1 in 8000) is it taken again in 64 bits (write_codes).  Rows of more than 16384 values, and rows whose
// numbers leave fp32's middle range, go through 64-bit loops (slow_row).
//
// Measured on a B200, L2 cold, beside the bytes at 6550 GB/s (us): quantise 32768 x 4096 bf16 66.3 (61.5), 2560 x 5120 fp32 10.8
// (10.0), read back 32768 x 4096 bf16 62.6 (61.5); norm 32768 x 2048 bf16 + fp32 stream 113 (113), fp32 + fp32 130 (133), bf16
// + bf16 82 (72), bf16 alone 68 (31): where few bytes come for each value, a norm is bound by its instructions (25 a value, issued
// in 74% of the cycles).  Odd widths, 20000 x 1111 bf16: quantise 29 (10), norm with an fp32 stream 89 (37).
#include <type_traits>
#include "int8_linear.cuh"

namespace mtp {
namespace {

using i8::MAX_COLS;

constexpr int MAX_HELD = 16384;        // columns of a row that a CTA holds
constexpr int LONG_THREADS = 256;
constexpr int UNROLL = 4;              // vectors that a thread reads back, their loads in flight together
constexpr float MAGIC = 12582912.f;    // 1.5 * 2^23: x + MAGIC is x rounded to a whole number, its low byte the int8
constexpr float BORDER = 0.5f - 1.f / 16384.f;
constexpr float FLT_TOP = 3.402823466e38f;
constexpr uint32_t TINY = 0x0d800000u, HUGE_ = 0x71800000u;  // 2^-100, 2^100

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }

// a / 127 rounded to nearest, by a product with 1 / 127 and a correction from its remainder (P. Markstein, IBM J. Res. Dev. 34,
// 1990: with 1 / b rounded to nearest and q within a unit in the last place, fma(a - q b, 1 / b, q) is the rounded quotient).
// With a division the norm is slower (32768 x 2048 bf16 alone: 70 us, 80), with the product alone a scale in 10^11 is
// another fp32 number.
__device__ __forceinline__ double over_127(double a) {
  constexpr double k = 1.0 / 127.0;
  const double q = __dmul_rn(a, k);
  return fma(fma(-127.0, q, a), k, q);
}

// fp32 scale of a row whose largest |y| is amax; NaN for a row with a NaN or an infinity (`bad`).
__device__ __forceinline__ float scale_of(double amax, bool bad) {
  const float s = (float)over_127(fmax(amax, 1e-8));
  return bad || !(s <= FLT_TOP) ? nan_f() : s;
}

__device__ __forceinline__ int exact_code(double y, float s) { return (int)fmin(fmax(rint(y / (double)s), -127.0), 127.0); }

// Codes of four values p * c, the quotients to fp32's precision: the codes in one word, and the largest distance from a code.
__device__ __forceinline__ uint32_t codes4(const float *p, float c, float &far) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = fmaf(p[i], c, MAGIC);
    far = fmaxf(far, fabsf(fmaf(p[i], c, -__fsub_rn(m[i], MAGIC))));
  }
  const uint32_t lo = __byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// Codes of four values x that are held exactly, k being 1 / s to fp32's precision.  x - q s is exact in fp32: a multiple of
// s's last place, and no more than about s / 2.  So q is the nearest where that is below s / 2, and else the one beside it,
// or in a tie the even one.  (A tie is no rarity among 16-bit values: half the largest of a row is one.)
__device__ __forceinline__ uint32_t exact_codes4(const float *x, float k, float s) {
  float m[4], rem[4], far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = fmaf(x[i], k, MAGIC);
    rem[i] = fmaf(-__fsub_rn(m[i], MAGIC), s, x[i]);
    far = fmaxf(far, fabsf(rem[i]));
  }
  const float half = 0.5f * s;
  if (far >= half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = fabsf(rem[i]);
      if (a > half || (a == half && (__float_as_uint(m[i]) & 1))) m[i] += copysignf(1.f, rem[i]);
    }
  }
  const uint32_t lo = __byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// x in 64 bits, converted where it stands: what is rarely needed shall not be kept from an earlier conversion.
__device__ __forceinline__ double widen(float x) {
  double d;
  asm volatile("cvt.f64.f32 %0, %1;" : "=d"(d) : "f"(x));
  return d;
}

// The code of a y whose quotient t = y / s (to fp32's precision) lies next to k + 1/2: s (k + 1/2) is exact in 64 bits.
__device__ __forceinline__ int border_code(double y, float t, float s) {
  const float k = floorf(t);
  const double e = ((double)k + 0.5) * (double)s;
  const int lo = (int)k;
  return y > e ? lo + 1 : y < e ? lo : lo + (lo & 1);
}

// ------------------------------------------------------------------ element access
// N values from p on: one or two vector loads, converted to fp32.
template <typename T, int N> struct Raw { uint32_t w[sizeof(T) * N / 4]; };

template <typename T, int N>
__device__ __forceinline__ void load_raw(Raw<T, N> &r, const T *p) {
  constexpr int W = sizeof(T) * N / 4;
  if constexpr (W == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t *>(p);
  } else if constexpr (W == 2) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    r.w[0] = u.x; r.w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4 *>(p + i * 4 / sizeof(T));
      r.w[i] = u.x; r.w[i + 1] = u.y; r.w[i + 2] = u.z; r.w[i + 3] = u.w;
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_raw(T *p, const Raw<T, N> &r) {
  constexpr int W = sizeof(T) * N / 4;
  if constexpr (W == 1) {
    *reinterpret_cast<uint32_t *>(p) = r.w[0];
  } else if constexpr (W == 2) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      *reinterpret_cast<uint4 *>(p + i * 4 / sizeof(T)) = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
  }
}
// N values of a row from column col on, wherever the row begins, zeros from column cols on: the aligned vector that the first
// of them lies in, and the next one if they reach into it, shifted together.  What is read lies within vectors that hold a value
// of the row.
template <typename T, int N>
__device__ __forceinline__ void load_ragged(Raw<T, N> &r, const T *row, int col, int cols) {
  constexpr int B = sizeof(T) * N, W = B / 4;
  static_assert(W <= 4, "what follows shifts by 8, 4, 2 and 1 bytes");
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + col), a = at & ~(uintptr_t)(B - 1);
  const uint32_t s = (uint32_t)(at - a);
  load_raw(r, reinterpret_cast<const T *>(a));
  if (s) {
    Raw<T, N> next{};
    if (a + B < reinterpret_cast<uintptr_t>(row + cols)) load_raw(next, reinterpret_cast<const T *>(a + B));
    uint32_t w[2 * W + 1];
#pragma unroll
    for (int i = 0; i < W; ++i) { w[i] = r.w[i]; w[W + i] = next.w[i]; }
    w[2 * W] = 0;
    if (W == 4 && (s & 8)) {
#pragma unroll
      for (int i = 0; i + 2 <= 2 * W; ++i) w[i] = w[i + 2];
    }
    if (W >= 2 && (s & 4)) {
#pragma unroll
      for (int i = 0; i + 1 <= 2 * W; ++i) w[i] = w[i + 1];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (s & 3));
  }
  const int n = cols - col;
  if (n < N) {
    constexpr int E = 4 / (int)sizeof(T);  // values in a word
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int in = n - i * E;  // of word i
      if (in <= 0) r.w[i] = 0;
      else if (in < E) r.w[i] &= (1u << (32 / E * in)) - 1u;
    }
  }
}
template <typename T, int N> __device__ __forceinline__ void store_ragged(T *row, int col, int cols, const Raw<T, N> &r) {
  T *to = row + col;
  const int n = cols - col;
  if (n >= N && (reinterpret_cast<uintptr_t>(to) & (sizeof(T) * N - 1)) == 0) {
    store_raw(to, r);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= n) continue;
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(to)[i] = r.w[i];
      else if constexpr (sizeof(T) == 2) reinterpret_cast<unsigned short *>(to)[i] = (unsigned short)(r.w[i / 2] >> (16 * (i & 1)));
      else to[i] = (T)(r.w[i / 4] >> (8 * (i & 3)));
    }
  }
}

template <typename T, int N> __device__ __forceinline__ void to_f32(const Raw<T, N> &r, float *v) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      v[i] = __uint_as_float(r.w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      v[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    } else {
      v[i] = __half2float(__ushort_as_half((unsigned short)(r.w[i / 2] >> (16 * (i & 1)))));
    }
  }
}
template <typename T, int N> __device__ __forceinline__ void from_f32(Raw<T, N> &r, const float *v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i], v[i + 1]);
        r.w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[i], v[i + 1]);
        r.w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  }
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
template <typename T> struct Code;
template <> struct Code<float> { static constexpr int value = MTP_F32; };
template <> struct Code<__nv_bfloat16> { static constexpr int value = MTP_BF16; };
template <> struct Code<__half> { static constexpr int value = MTP_F16; };

// The largest of m, |a| and |b|; NaN if one is.
__device__ __forceinline__ float max_abs3(float m, float a, float b) {
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
  return m;
}

// ------------------------------------------------------------------ teams
struct Join {
  double d[32];
  uint32_t u[32];
  unsigned long long most;
};

// A warp or a CTA.  Every thread of the team calls each of these.
template <bool WARP> struct Team {
  Join *j;
  __device__ __forceinline__ int rank() const { return WARP ? threadIdx.x & 31 : threadIdx.x; }
  __device__ __forceinline__ int size() const { return WARP ? 32 : blockDim.x; }
  __device__ __forceinline__ void sync() const {
    if (WARP) __syncwarp();
    else __syncthreads();
  }
  __device__ __forceinline__ uint32_t max_u32(uint32_t v) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) j->u[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5, lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < n ? j->u[lane] : 0u);
  }
  // The sum of s in a fixed order and the largest u.
  __device__ __forceinline__ void sum_max(double &s, uint32_t &u) const {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    u = __reduce_max_sync(0xffffffffu, u);
    if (WARP) return;
    const int n = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (n == 1) {
      __syncwarp();  // what one lane has set up for the team
      return;
    }
    if (lane == 0) {
      j->d[threadIdx.x >> 5] = s;
      j->u[threadIdx.x >> 5] = u;
    }
    __syncthreads();
    s = lane < n ? j->d[lane] : 0.0;
    u = __reduce_max_sync(0xffffffffu, lane < n ? j->u[lane] : 0u);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  // The largest of values that are not negative; few threads have one above 0.  `most` is 0 before the first call and is not
  // used twice between barriers.
  __device__ __forceinline__ double max_rare(double v) const {
    if (WARP) {
#pragma unroll
      for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
      return v;
    }
    if (v > 0.0) atomicMax(&j->most, (unsigned long long)__double_as_longlong(v));  // ordered as their bits are
    __syncthreads();
    return __longlong_as_double((long long)j->most);
  }
  __device__ __forceinline__ double max_all(double v) const {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (WARP) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) j->d[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) v = fmax(v, j->d[i]);
    return v;
  }
};

// A row in 64 bits throughout: h[c] is read from memory, y = h * rs * w (w NULL: y = h).  For long rows, and for rows whose
// numbers leave fp32's middle range.
template <bool WARP>
__device__ __noinline__ void slow_row(const Team<WARP> &team, const void *h, int h_dtype, const void *w, int w_dtype, double rs,
                                      int cols, int8_t *codes, float *scale) {
  double amax = 0.0;
  uint32_t bad = 0;
  for (int c = team.rank(); c < cols; c += team.size()) {
    double y = (double)ld_any(h, h_dtype, c);
    if (w) y = y * rs * (double)ld_any(w, w_dtype, c);
    y = fabs(y);
    bad |= !(y <= 1e300);
    amax = fmax(amax, y);
  }
  amax = team.max_all(amax);
  team.sync();
  const float s = scale_of(amax, team.max_u32(bad) != 0);
  for (int c = team.rank(); c < cols; c += team.size()) {
    double y = (double)ld_any(h, h_dtype, c);
    if (w) y = y * rs * (double)ld_any(w, w_dtype, c);
    codes[c] = (int8_t)(s > 0.f ? exact_code(y, s) : 0);
  }
  if (team.rank() == 0) *scale = s;
}

// The vectors of a row that a thread holds: those at columns (v * size + rank) * VEC.
template <int VEC, bool RAGGED, int NV, typename T>
__device__ __forceinline__ void load_row(Raw<T, VEC> (&raw)[NV], const T *row, int cols, int rank, int size) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = (v * size + rank) * VEC;
    if (col >= cols) raw[v] = Raw<T, VEC>{};
    else if (RAGGED) load_ragged(raw[v], row, col, cols);
    else load_raw(raw[v], row + col);
  }
}

// Writes the codes of the values that a thread holds, four to a word.
template <int VEC, bool RAGGED, int EACH>
__device__ __forceinline__ void store_codes(const uint32_t (&q)[EACH / 4], int8_t *codes, int cols, int rank, int size) {
#pragma unroll
  for (int v = 0; v < EACH / VEC; ++v) {
    const int col = (v * size + rank) * VEC;
    if (col >= cols) continue;
    Raw<int8_t, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) r.w[i] = q[v * (VEC / 4) + i];
    if (RAGGED) store_ragged(codes, col, cols, r);
    else store_raw(codes + col, r);
  }
}

// Writes the codes of the products p[] * c that a thread holds; value(i, col) gives the i-th's y in 64 bits.  INLINE: where it
// takes its values from registers, each border stands on its own; else they are met in a loop after the words are written, which
// keeps the kernel's code short (32768 x 1024 bf16 alone 38 us, each on its own 46).
template <int VEC, bool RAGGED, int EACH, bool INLINE, typename Y>
__device__ __forceinline__ void write_codes(const float (&p)[EACH], float c, float s, int8_t *codes, int cols, int rank, int size,
                                            Y value) {
  uint32_t q[EACH / 4], near[(EACH + 31) / 32] = {};
#pragma unroll
  for (int g = 0; g < EACH / 4; ++g) {
    float far = 0.f;
    q[g] = codes4(p + 4 * g, c, far);
    if (far > BORDER) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = 4 * g + k;
        const float m = fmaf(p[i], c, MAGIC);
        if (fabsf(fmaf(p[i], c, -__fsub_rn(m, MAGIC))) > BORDER) {
          if (INLINE) {
            const int col = ((i / VEC) * size + rank) * VEC + i % VEC;
            const uint32_t code = (uint32_t)border_code(value(i, col), __fmul_rn(p[i], c), s) & 0xffu;
            q[g] = (q[g] & ~(0xffu << (8 * k))) | code << (8 * k);
          } else {
            near[i / 32] |= 1u << (i & 31);
          }
        }
      }
    }
  }
  store_codes<VEC, RAGGED, EACH>(q, codes, cols, rank, size);
  if (!INLINE) {
#pragma unroll
    for (int j = 0; j < (EACH + 31) / 32; ++j) {
#pragma unroll 1
      for (uint32_t left = near[j]; left; left &= left - 1) {
        const int i = 32 * j + __ffs(left) - 1, col = ((i / VEC) * size + rank) * VEC + i % VEC;
        const double y = value(i, col);
        codes[col] = (int8_t)border_code(y, (float)(y / (double)s), s);
      }
    }
  }
}

// ------------------------------------------------------------------ quantise
template <typename T, int VEC, bool RAGGED, int EACH, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : (MAX_HELD / EACH + 31) / 32 * 32)
    quantize_kernel(const T *__restrict__ x, int64_t ld, int64_t rows, int cols, int8_t *__restrict__ codes, int64_t ld_codes,
                    float *__restrict__ scale) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ Join join;
  const Team<WARP> team{&join};
  const int rank = team.rank(), size = team.size();
  const int64_t r = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (r >= rows) return;
  const T *xr = x + r * ld;
  float p[EACH];
  Raw<T, VEC> raw[EACH / VEC];
  load_row<VEC, RAGGED>(raw, xr, cols, rank, size);
#pragma unroll
  for (int v = 0; v < EACH / VEC; ++v) to_f32(raw[v], p + v * VEC);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; i += 2) m = max_abs3(m, p[i], p[i + 1]);
  const uint32_t bits = team.max_u32(__float_as_uint(m));  // as integers: NaN above infinity above all numbers
  m = __uint_as_float(bits);
  const float s = bits >= 0x7f800000u ? nan_f() : __fdiv_rn(fmaxf(m, 1e-8f), 127.f);
  int8_t *out = codes + r * ld_codes;
  if (!(s > 0.f)) {
    for (int c = rank; c < cols; c += size) out[c] = 0;
  } else {
    const float k = __frcp_rn(s);  // 3.7e-37 at least: a normal number
    uint32_t q[EACH / 4];
#pragma unroll
    for (int i = 0; i < EACH; i += 4) q[i / 4] = exact_codes4(p + i, k, s);
    store_codes<VEC, RAGGED, EACH>(q, out, cols, rank, size);
  }
  if (rank == 0) scale[r] = s;
}

template <typename T>
__global__ void __launch_bounds__(LONG_THREADS) quantize_long_kernel(const T *x, int64_t ld, int64_t rows, int cols, int8_t *codes,
                                                                     int64_t ld_codes, float *scale) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ Join join;
  const Team<false> team{&join};
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    slow_row(team, x + r * ld, Code<T>::value, nullptr, 0, 1.0, cols, codes + r * ld_codes, scale + r);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ norm
struct NormArgs {
  const void *x, *resid;
  void *r_out;
  const void *w;
  int64_t ld_x, ld_r, ld_ro;
  int64_t rows;
  int cols, x_dtype, r_dtype, w_dtype;
  float eps;
  int8_t *codes;
  int64_t ld_codes;
  float *scale;
  double inv_cols;
};

template <int VEC, bool RAGGED, typename T>
__device__ __forceinline__ void load_weight_of(const T *w, int col, int cols, float *v) {
  if constexpr (RAGGED && sizeof(T) * VEC > 16) {
    // 8 fp32 weights beside 16-bit rows: 32 bytes, more than load_ragged shifts together.  As two vectors where the weight lies on
    // 16-byte boundaries, as an allocation does (20000 x 1111 fp16 + fp16: 74 us), else one by one (88).
    if ((reinterpret_cast<uintptr_t>(w) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        Raw<T, 4> r{};
        if (col + i < cols) load_raw(r, w + col + i);
        to_f32(r, v + i);
      }
#pragma unroll
      for (int i = 1; i < VEC; ++i)
        if (col + i >= cols) v[i] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = col + i < cols ? ldf(w + col + i) : 0.f;
    }
  } else {
    Raw<T, VEC> r;
    if constexpr (RAGGED) load_ragged(r, w, col, cols);
    else load_raw(r, w + col);
    to_f32(r, v);
  }
}
template <int VEC, bool RAGGED>
__device__ __forceinline__ void load_weight(const void *w, int dtype, int col, int cols, float *v) {
  if (dtype == MTP_F32) load_weight_of<VEC, RAGGED>((const float *)w, col, cols, v);
  else if (dtype == MTP_BF16) load_weight_of<VEC, RAGGED>((const __nv_bfloat16 *)w, col, cols, v);
  else load_weight_of<VEC, RAGGED>((const __half *)w, col, cols, v);
}

struct None {};

// TR is the residual's type, or None.  y = h w r with r = 1 / sqrt(mean h^2 + eps); the scale is fp32(max |y| / 127), and the
// codes are those of (h w) (r / scale).  The sum of squares and r are held in 64 bits; the largest product is found among the
// fp32 products and then taken exactly (a 48-bit number) from the values whose product rounds to that.
template <typename TX, typename TR, int VEC, bool RAGGED, int EACH, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : EACH == 8 ? 1024 : (MAX_HELD / EACH + 31) / 32 * 32) norm_kernel(const NormArgs a) {
  constexpr bool ADD = !std::is_same<TR, None>::value;
  constexpr bool KEEP = EACH == 8;  // few rows: h stays in registers, where else a value of it is read again if need be
  using TH = typename std::conditional<ADD, TR, TX>::type;  // the stream's type
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ Join join;
  const Team<WARP> team{&join};
  const int rank = team.rank(), size = team.size(), cols = a.cols;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;
  if (!WARP && threadIdx.x == 0) join.most = 0;  // the first use comes after the barrier of sum_max
  const TX *xr = (const TX *)a.x + row * a.ld_x;
  const TR *rr = (const TR *)a.resid + row * a.ld_r;
  TR *ro = (TR *)a.r_out + row * a.ld_ro;
  constexpr int NV = EACH / VEC;
  float p[EACH], w[EACH];
  Raw<TX, VEC> raw[NV];
  load_row<VEC, RAGGED>(raw, xr, cols, rank, size);
  if constexpr (ADD) {
    Raw<TR, VEC> res[NV];
    load_row<VEC, RAGGED>(res, rr, cols, rank, size);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * size + rank) * VEC;
      float f[VEC], h[VEC];
      to_f32(raw[v], f);
      to_f32(res[v], h);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = __fadd_rn(f[i], h[i]);
      from_f32(res[v], h);
      to_f32(res[v], p + v * VEC);  // as it is held
      if (col < cols) {
        if (RAGGED) store_ragged(ro, col, cols, res[v]);
        else store_raw(ro + col, res[v]);
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) to_f32(raw[v], p + v * VEC);
  }
  auto weights = [&] {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = (v * size + rank) * VEC;
      if (col < cols) {
        load_weight<VEC, RAGGED>(a.w, a.w_dtype, col, cols, w + v * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[v * VEC + i] = 0.f;
      }
    }
  };
  if (!RAGGED) weights();  // ragged rows have the registers of their shifts to themselves first (20000 x 1111 bf16 + fp32: 88 us, else 98)
  double ss = 0.0, ss2 = 0.0;
  float top_here = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; i += 2) {
    const double h0 = (double)p[i], h1 = (double)p[i + 1];
    ss = fma(h0, h0, ss);
    ss2 = fma(h1, h1, ss2);
  }
  ss += ss2;
  if (RAGGED) weights();
  float h[KEEP ? EACH : 1];
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (KEEP) h[i] = p[i];
#pragma unroll
  for (int i = 0; i < EACH; i += 2) {
    p[i] = __fmul_rn(p[i], w[i]);
    p[i + 1] = __fmul_rn(p[i + 1], w[i + 1]);
    top_here = max_abs3(top_here, p[i], p[i + 1]);
  }
  const uint32_t mine = __float_as_uint(top_here);  // as integers: NaN above infinity above all numbers
  uint32_t most = mine;
  team.sum_max(ss, most);
  const double rs = rsqrt(fma(ss, a.inv_cols, (double)a.eps));
  const void *hp = ADD ? (const void *)ro : (const void *)xr;  // a thread reads back only what it has stored itself
  auto y_of = [&](int i, int col) {
    if constexpr (KEEP) return widen(h[i]) * rs * widen(w[i]);
    else return (double)ldf((const TH *)hp + col) * rs * (double)ld_any(a.w, a.w_dtype, col);
  };
  int8_t *out = a.codes + row * a.ld_codes;
  if (most >= TINY && most <= HUGE_ && rs < 1e30) {
    double top = 0.0;
    uint32_t at_top[(EACH + 31) / 32] = {};
    if (mine == most) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        if ((__float_as_uint(p[i]) & 0x7fffffffu) == most) {
          const int col = ((i / VEC) * size + rank) * VEC + i % VEC;
          if (KEEP) top = fmax(top, fabs(y_of(i, col)));
          else at_top[i / 32] |= 1u << (i & 31);
        }
      }
    }
    if (!KEEP) {
#pragma unroll
      for (int j = 0; j < (EACH + 31) / 32; ++j) {
#pragma unroll 1
        for (uint32_t left = at_top[j]; left; left &= left - 1) {
          const int i = 32 * j + __ffs(left) - 1, col = ((i / VEC) * size + rank) * VEC + i % VEC;
          top = fmax(top, fabs(y_of(i, col)));
        }
      }
    }
    top = team.max_rare(top);
    const float s = scale_of(top, false);
    const float c = __fmul_rn((float)rs, __frcp_rn(s));  // NaN, and so not taken, where s is not finite
    const uint32_t cb = __float_as_uint(c);
    if (cb >= TINY && cb <= HUGE_) {
      write_codes<VEC, RAGGED, EACH, KEEP>(p, c, s, out, cols, rank, size, y_of);
      if (rank == 0) a.scale[row] = s;
      return;
    }
  }
  team.sync();  // what other threads of the team have stored of the row
  slow_row(team, hp, Code<TH>::value, a.w, a.w_dtype, rs, cols, out, a.scale + row);
}

__global__ void __launch_bounds__(LONG_THREADS) norm_long_kernel(const NormArgs a) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ Join join;
  const Team<false> team{&join};
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    double ss = 0.0;
    uint32_t none = 0;
    for (int c = threadIdx.x; c < a.cols; c += LONG_THREADS) {
      float h = ld_any(a.x, a.x_dtype, r * a.ld_x + c);
      if (a.resid) h = st_any(a.r_out, a.r_dtype, r * a.ld_ro + c, __fadd_rn(h, ld_any(a.resid, a.r_dtype, r * a.ld_r + c)));
      ss = fma((double)h, (double)h, ss);
    }
    team.sum_max(ss, none);
    const double rs = rsqrt(fma(ss, a.inv_cols, (double)a.eps));
    const int h_dtype = a.resid ? a.r_dtype : a.x_dtype;
    const char *h = (const char *)(a.resid ? a.r_out : a.x) + r * (a.resid ? a.ld_ro : a.ld_x) * (h_dtype == MTP_F32 ? 4 : 2);
    slow_row(team, h, h_dtype, a.w, a.w_dtype, rs, a.cols, a.codes + r * a.ld_codes, a.scale + r);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ read back
// A thread takes N codes of a row and writes 16 bytes (N = 1: rows of any alignment).
template <typename T, int N, typename I>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t *__restrict__ codes, int64_t ld_codes,
                                                         const float *__restrict__ scale, T *__restrict__ out, int64_t ld_out,
                                                         I parts, I per_row) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  uint32_t w[UNROLL][N / 4 + (N == 1)];
  float s[UNROLL];
  T *to[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const I i = ((I)blockIdx.x * UNROLL + u) * 256 + threadIdx.x;
    to[u] = nullptr;
    if (i < parts) {
      const I r = i / per_row;
      const int c = (int)(i - r * per_row) * N;
      const int8_t *from = codes + (int64_t)r * ld_codes + c;
      to[u] = out + (int64_t)r * ld_out + c;
      s[u] = scale[r];
      if constexpr (N == 1) {
        w[u][0] = (uint8_t)*from;
      } else if constexpr (N == 4) {
        w[u][0] = *reinterpret_cast<const uint32_t *>(from);
      } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(from);
        w[u][0] = v.x; w[u][1] = v.y;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (!to[u]) continue;
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __fmul_rn((float)(int8_t)(w[u][k / 4] >> (8 * (k & 3))), s[u]);
    if constexpr (N == 1) {
      stf(to[u], v[0]);
    } else {
      Raw<T, N> raw;
      from_f32(raw, v);
      store_raw(to[u], raw);
    }
  }
}

// Dense results of rows of any alignment: a thread takes N values of them that lie in 16 bytes, of one row or of several.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_dense_kernel(const int8_t *__restrict__ codes, int64_t ld_codes,
                                                               const float *__restrict__ scale, T *__restrict__ out, int64_t total,
                                                               int cols) {
  constexpr int N = 16 / (int)sizeof(T);
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t at = (((int64_t)blockIdx.x * UNROLL + u) * 256 + threadIdx.x) * N;
    if (at >= total) return;
    int64_t r = at <= 0x7fffffff ? (int64_t)((uint32_t)at / (uint32_t)cols) : at / cols;
    int c = (int)(at - r * cols);
    float v[N];
    if (c + N <= cols) {
      Raw<int8_t, N> q;
      load_ragged(q, codes + r * ld_codes, c, cols);
      const float s = scale[r];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = __fmul_rn((float)(int8_t)(q.w[k / 4] >> (8 * (k & 3))), s);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v[k] = at + k < total ? __fmul_rn((float)codes[r * ld_codes + c], scale[r]) : 0.f;
        if (++c == cols) { c = 0; ++r; }
      }
    }
    Raw<T, N> raw;
    from_f32(raw, v);
    if (at + N <= total) {
      store_raw(out + at, raw);
    } else {
      for (int k = 0; at + k < total; ++k) stf(out + at + k, v[k]);
    }
  }
}

template <typename T, int N>
void launch_dequantize(const int8_t *codes, int64_t ld_codes, const float *scale, int64_t rows, int cols, T *out, int64_t ld_out,
                       cudaStream_t s) {
  const int64_t per_row = cols / N, parts = rows * per_row;
  const dim3 grid((unsigned)((parts + 256 * UNROLL - 1) / (256 * UNROLL)));
  if (parts < 0x7fff0000)
    launch_pdl(dequantize_kernel<T, N, uint32_t>, grid, dim3(256), 0, s, codes, ld_codes, scale, out, ld_out, (uint32_t)parts,
               (uint32_t)per_row);
  else
    launch_pdl(dequantize_kernel<T, N, int64_t>, grid, dim3(256), 0, s, codes, ld_codes, scale, out, ld_out, parts, per_row);
}

// ------------------------------------------------------------------ host side
bool dtype_ok(int d) { return d == MTP_F32 || d == MTP_BF16 || d == MTP_F16; }
bool rows_ok(int64_t rows, int cols) { return rows >= 0 && rows <= 0x7fffffffll && cols >= 1 && cols <= MAX_COLS; }
int size_of(int dtype) { return dtype == MTP_F32 ? 4 : 2; }

// Rows from p on, ld elements of es bytes apart, in vectors of n.
bool on_vectors(const void *p, int64_t ld, int es, int64_t rows, int n) {
  return aligned(p, es * n < 16 ? es * n : 16) && (rows == 1 || ld * es % (es * n < 16 ? es * n : 16) == 0);
}

// Rows of up to 1024 values go to warps, eight to a CTA, with 16, 24 or 32 values a lane (60000 x 320 bf16 16.6 us, with 32 24.2; 32768
// x 768 14.1, with 32 16.0), many rows to 1536 with 48 (32768 x 1536 bf16 27.5 us, by CTAs 36.5; though not ragged ones: 1335 fp32
// 94 and 78), longer ones to CTAs of as many threads as hold them.
template <typename T, int VEC, bool RAGGED, int EACH, bool WARP>
void launch_quantize_team(const T *x, int64_t ld, int64_t rows, int cols, int8_t *codes, int64_t ld_codes, float *scale,
                          cudaStream_t s) {
  const unsigned grid = (unsigned)(WARP ? (rows + 7) / 8 : rows), threads = WARP ? 256 : ceil_div(cols, EACH * 32) * 32;
  launch_pdl(quantize_kernel<T, VEC, RAGGED, EACH, WARP>, dim3(grid), dim3(threads), 0, s, x, ld, rows, cols, codes, ld_codes, scale);
}

// A CTA has 32 values a thread where rows are many (32768 x 4096 bf16: 66.5 us, with 16 74.9), 16 where they are few and a
// row's own time counts (1 x 4096: 1.6 us, with 32 2.0).
template <typename T, int VEC, bool RAGGED>
void launch_quantize(const T *x, int64_t ld, int64_t rows, int cols, int8_t *codes, int64_t ld_codes, float *scale,
                     cudaStream_t s) {
  if (cols <= 512) launch_quantize_team<T, VEC, RAGGED, 16, true>(x, ld, rows, cols, codes, ld_codes, scale, s);
  else if (cols <= 768) launch_quantize_team<T, VEC, RAGGED, 24, true>(x, ld, rows, cols, codes, ld_codes, scale, s);
  else if (cols <= 1024) launch_quantize_team<T, VEC, RAGGED, 32, true>(x, ld, rows, cols, codes, ld_codes, scale, s);
  else if (rows <= 4 * num_sms()) launch_quantize_team<T, VEC, RAGGED, 16, false>(x, ld, rows, cols, codes, ld_codes, scale, s);
  else if (cols <= 1536 && !RAGGED) launch_quantize_team<T, VEC, false, 48, true>(x, ld, rows, cols, codes, ld_codes, scale, s);
  else launch_quantize_team<T, VEC, RAGGED, 32, false>(x, ld, rows, cols, codes, ld_codes, scale, s);
}

template <typename TX, typename TR, int VEC, bool RAGGED, int EACH, bool WARP> void launch_norm_kernel(const NormArgs &a, cudaStream_t s) {
  const unsigned grid = (unsigned)(WARP ? (a.rows + 7) / 8 : a.rows), threads = WARP ? 256 : ceil_div(a.cols, EACH * 32) * 32;
  launch_pdl(norm_kernel<TX, TR, VEC, RAGGED, EACH, WARP>, dim3(grid), dim3(threads), 0, s, a);
}

// A norm's rows of up to 768 values go to warps (60000 x 768 fp32: 92 us, by CTAs 95), longer ones to CTAs (32768 x 1024 fp32: 69 us,
// by warps 74; ragged, 1001: 128 and 209).  A CTA has 16 values a thread (32768 x 2048 bf16 + fp32: 113 us, with 32 135), but where x
// and the stream are of 16 bits and take few registers 24 or 32, whichever leaves fewer without a value (bf16 alone: 68 us, with 16
// 75; 1536 columns: 54, with 32 66), though not for ragged rows (20000 x 1111: 45 us, with 32 68).  Few rows have CTAs of 8 values a
// thread whatever their length (1 x 2048: 2.4 us, with 16 2.9).
template <typename TX, typename TR, int VEC, bool RAGGED> void launch_norm_team(const NormArgs &a, cudaStream_t s) {
  if (a.rows <= 4 * num_sms() && a.cols <= MAX_HELD / 2) launch_norm_kernel<TX, TR, VEC, RAGGED, 8, false>(a, s);
  else if (a.cols <= 512) launch_norm_kernel<TX, TR, VEC, RAGGED, 16, true>(a, s);
  else if (a.cols <= 768) launch_norm_kernel<TX, TR, VEC, RAGGED, 24, true>(a, s);
  else if constexpr (VEC == 4 || RAGGED) launch_norm_kernel<TX, TR, VEC, RAGGED, 16, false>(a, s);
  else if (ceil_div(a.cols, 768) * 768 < ceil_div(a.cols, 1024) * 1024) launch_norm_kernel<TX, TR, VEC, RAGGED, 24, false>(a, s);
  else launch_norm_kernel<TX, TR, VEC, RAGGED, 32, false>(a, s);
}

template <typename TX, typename TR> void launch_norm(const NormArgs &a, cudaStream_t s) {
  constexpr bool ADD = !std::is_same<TR, None>::value;
  constexpr bool WIDE = std::is_same<TX, float>::value || std::is_same<TR, float>::value;
  constexpr int VEC = WIDE ? 4 : 8;  // 16 bytes of the wider type
  const int er = size_of(a.r_dtype);
  const bool vec = a.cols % VEC == 0 && on_vectors(a.x, a.ld_x, sizeof(TX), a.rows, VEC) &&
                   on_vectors(a.w, 0, size_of(a.w_dtype), 1, VEC) && on_vectors(a.codes, a.ld_codes, 1, a.rows, VEC) &&
                   (!ADD || (on_vectors(a.resid, a.ld_r, er, a.rows, VEC) && on_vectors(a.r_out, a.ld_ro, er, a.rows, VEC)));
  if (vec) launch_norm_team<TX, TR, VEC, false>(a, s);
  else launch_norm_team<TX, TR, VEC, true>(a, s);
}

template <typename TX> bool launch_norm_of(const NormArgs &a, cudaStream_t s) {
  if (!a.resid) launch_norm<TX, None>(a, s);
  else if (a.r_dtype == MTP_F32) launch_norm<TX, float>(a, s);
  else if (!std::is_same<TX, float>::value && a.r_dtype == Code<TX>::value) launch_norm<TX, TX>(a, s);
  else return false;
  return true;
}

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
  MTP_REQUIRE(rows == 1 || (ld >= cols && ld_codes >= cols), "leading dimensions too small");
  cudaStream_t s = (cudaStream_t)stream;
  MTP_DISPATCH_3(dtype, T, {
    constexpr int VEC = sizeof(T) == 4 ? 4 : 8;
    if (cols > MAX_HELD)
      launch_pdl(quantize_long_kernel<T>, dim3((unsigned)(rows < 148 * 8 ? rows : 148 * 8)), dim3(LONG_THREADS), 0, s,
                 (const T *)x, ld, rows, cols, codes, ld_codes, scale);
    else if (cols % VEC == 0 && on_vectors(x, ld, sizeof(T), rows, VEC) && on_vectors(codes, ld_codes, 1, rows, VEC))
      launch_quantize<T, VEC, false>((const T *)x, ld, rows, cols, codes, ld_codes, scale, s);
    else
      launch_quantize<T, VEC, true>((const T *)x, ld, rows, cols, codes, ld_codes, scale, s);
  });
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
  MTP_DISPATCH_3(out_dtype, T, {
    constexpr int N = 16 / sizeof(T);
    if (cols % N == 0 && on_vectors(codes, ld_codes, 1, rows, N) && on_vectors(out, ld_out, sizeof(T), rows, N))
      launch_dequantize<T, N>(codes, ld_codes, scale, rows, cols, (T *)out, ld_out, s);
    else if (aligned16(out) && (rows == 1 || ld_out == cols))
      launch_pdl(dequantize_dense_kernel<T>, dim3((unsigned)((rows * cols + 256 * UNROLL * N - 1) / (256 * UNROLL * N))), dim3(256), 0,
                 s, codes, ld_codes, scale, (T *)out, rows * cols, cols);
    else
      launch_dequantize<T, 1>(codes, ld_codes, scale, rows, cols, (T *)out, ld_out, s);
  });
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
  const NormArgs a{x, resid, resid_out, w, ld_x, ld_resid, ld_resid_out, rows, cols, x_dtype, resid_dtype, w_dtype, eps, codes,
                   ld_codes, scale, 1.0 / cols};
  bool done = false;
  if (cols <= MAX_HELD) MTP_DISPATCH_3(x_dtype, T, done = launch_norm_of<T>(a, s));
  if (!done)  // long rows, and every 16-bit stream of another type than x, fp32 x with a 16-bit stream among them (598 us for 32768 x 2048)
    launch_pdl(norm_long_kernel, dim3((unsigned)(rows < 148 * 8 ? rows : 148 * 8)), dim3(LONG_THREADS), 0, s, a);
  return check_launch("rmsnorm_int8");
}

}  // extern "C"

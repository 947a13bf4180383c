// Softmax statistics shared by the kernels over logits rows and the lm_head kernel that never writes logits.
#pragma once
#include "common.cuh"

namespace mtp {
namespace lg {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3.402823466e38f;
constexpr float FLOOR_Y = -1024.f;  // 2^FLOOR_Y is 0: stands for -inf where it is multiplied by a 0

// ----------------------------------------------------------------- arithmetic
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Packed fp32 pairs (one instruction for two lanes' worth of arithmetic).
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(F2 p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// ----------------------------------------------------------------- row statistics
// Of a set of elements: m their largest (LOWEST if they are none or all -inf: then s is 0), s = sum e^((x - m) / T),
// u = sum e^y y with y = (x - m) / T * log2 e.  A NaN or +inf among them makes s NaN.
struct Stat {
  float m, s, u;
};

template <bool ENT>
__device__ __forceinline__ Stat join(Stat a, Stat b, float c2) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  const float ya = fmaxf((a.m - r.m) * c2, FLOOR_Y), yb = fmaxf((b.m - r.m) * c2, FLOOR_Y);
  const float ea = ex2(ya), eb = ex2(yb);
  r.s = a.s * ea + b.s * eb;
  r.u = ENT ? fmaf(ya, a.s, a.u) * ea + fmaf(yb, b.s, b.u) * eb : 0.f;
  return r;
}

// Adds N elements; returns the largest of each half of them (NaN passed over).  masked: a logit of -inf (or NaN) has been
// met, whose e^y y is 0 * -inf; found by the sum turning NaN, which costs one comparison where there are none.  MASKED:
// there may be more, so that y is kept at FLOOR_Y or above.
template <bool ENT, int N, bool MASKED = false>
__device__ __forceinline__ float2 accumulate(Stat &st, const float (&x)[N], float c2, bool &masked) {
  float2 mx = make_float2(x[0], x[N / 2]);
#pragma unroll
  for (int i = 1; i + 1 < N / 2; i += 2) {
    mx.x = max3(mx.x, x[i], x[i + 1]);
    mx.y = max3(mx.y, x[N / 2 + i], x[N / 2 + i + 1]);
  }
  if (N / 2 % 2 == 0) {
    mx.x = fmaxf(mx.x, x[N / 2 - 1]);
    mx.y = fmaxf(mx.y, x[N - 1]);
  }
  const float m = max3(st.m, mx.x, mx.y);
  const float dy = fmaxf((st.m - m) * c2, FLOOR_Y);
  const float corr = ex2(dy);
  const F2 nm = f2(-m, -m), cc = f2(c2, c2);
  F2 s = f2(0.f, 0.f), u = f2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const F2 y = mul2(add2(f2(x[i], x[i + 1]), nm), cc);
    float y0, y1;
    un2(y, y0, y1);
    const F2 e = f2(ex2(y0), ex2(y1));
    s = add2(s, e);
    if constexpr (ENT) u = fma2(e, MASKED ? f2(fmaxf(y0, FLOOR_Y), fmaxf(y1, FLOOR_Y)) : y, u);
  }
  float s0, s1;
  un2(s, s0, s1);
  if constexpr (ENT) {
    float u0, u1;
    un2(u, u0, u1);
    u0 += u1;
    if (!MASKED && u0 != u0) {  // the same with y no lower than FLOOR_Y
      masked = true;
      u0 = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float y = (x[i] - m) * c2;
        u0 = fmaf(ex2(y), fmaxf(y, FLOOR_Y), u0);
      }
    }
    st.u = fmaf(fmaf(dy, st.s, st.u), corr, u0);
  }
  st.s = fmaf(st.s, corr, s0 + s1);
  st.m = m;
  return mx;
}

template <bool ENT>
__device__ __forceinline__ void accumulate1(Stat &st, float x, float c2) {
  const float v[2] = {x, -INFINITY};
  bool masked;
  accumulate<ENT, 2, true>(st, v, c2, masked);
}

struct RowStats {
  float m, log_s, entropy;  // m: largest logit (not divided by T), -inf for a row of -inf alone
};

__device__ __forceinline__ RowStats finish(Stat st) {
  if (st.s == 0.f) return {-INFINITY, 0.f, 0.f};
  const float ls = logf(st.s);
  return {st.m, ls, ls - LN2 * (st.u / st.s)};
}

// Of a row whose logits are not to be trusted, because a device wait of the pass that made them expired: everything that
// is derived from it is NaN (a largest logit of -inf would give log probabilities of -inf, as of a row of -inf alone).
__device__ __forceinline__ RowStats expired() { return {NAN, NAN, NAN}; }

// log p of a logit of the row; a row whose logits are all -inf gives -inf.
__device__ __forceinline__ float log_prob(float x, float m, float log_s, float inv_t) {
  return m == -INFINITY ? -INFINITY : (x - m) * inv_t - log_s;
}

}  // namespace lg
}  // namespace mtp

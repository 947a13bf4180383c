// Operators on logits rows: the log probability of a given token with entropy and top alternatives, its gradient, and
// the distillation loss from a teacher's top logits with its gradient.
//
// With z = x / T, m = max z and S = sum e^(z - m), a row gives
//   log p_j = (z_j - m) - log S          H = log S - sum e^(z - m) (z - m) / S
// All sums and statistics are fp32.  One CTA per row.
#include "common.cuh"

namespace mtp {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_TOP = 128;  // alternatives or teacher entries per row
constexpr int NT = 256;

// Row r of a batch laid out as [outer][inner] rows: r = o * inner + i.
struct Rows {
  int64_t inner, ld_outer, ld;
  __device__ __forceinline__ int64_t at(int64_t r) const { return (r / inner) * ld_outer + (r % inner) * ld; }
};

// Order of the alternatives as unsigned integers: larger value first, -0 equal to +0, NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = v == 0.f ? 0u : __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float nan_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename F, typename T>
__device__ __forceinline__ T block_reduce(T v, T *red, F op) {
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  T s = red[0];
  for (int i = 1; i < NT / 32; ++i) s = op(s, red[i]);  // fixed order: the same in every thread
  return s;
}

__device__ __forceinline__ float sum_op(float a, float b) { return a + b; }

struct RowStats {
  float m, log_s, entropy;  // m: largest logit (not divided by T)
};

// log p of a logit of the row; a row whose logits are all -inf gives -inf.
__device__ __forceinline__ float log_prob(float x, float m, float log_s, float inv_t) {
  return m == -INFINITY ? -INFINITY : (x - m) * inv_t - log_s;
}

template <typename T>
__device__ RowStats row_stats(const T *row, int V, float inv_t, float *red) {
  auto fmx = [](float a, float b) { return nan_max(a, b); };
  auto add = [](float a, float b) { return sum_op(a, b); };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += NT) m = nan_max(m, ldf(row + i));
  m = block_reduce(m, red, fmx);
  if (m == -INFINITY) return {m, 0.f, 0.f};
  float s = 0.f, u = 0.f;
  for (int i = threadIdx.x; i < V; i += NT) {
    const float d = (ldf(row + i) - m) * inv_t;
    const float e = expf(d);
    s += e;
    u += e * fmaxf(d, -1000.f);  // e is 0 below: a masked logit adds nothing
  }
  s = block_reduce(s, red, add);
  u = block_reduce(u, red, add);
  const float ls = logf(s);
  return {m, ls, ls - u / s};
}

struct FwdArgs {
  const int64_t *targets;
  float *logprob, *entropy, *stats;
  int top_k;
  int64_t *top_ids;
  float *top_logprobs;
  float inv_t;
  int V;
};

template <typename T>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const T *__restrict__ logits, Rows rows, FwdArgs a) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ float red[NT / 32];
  __shared__ unsigned long long redk[NT / 32];
  const int64_t r = blockIdx.x;
  const T *row = logits + rows.at(r);
  const RowStats st = row_stats(row, a.V, a.inv_t, red);
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int64_t t = a.targets[r];
      a.logprob[r] = t < 0 ? 0.f : t >= a.V ? NAN : log_prob(ldf(row + t), st.m, st.log_s, a.inv_t);
    }
    if (a.entropy) a.entropy[r] = st.entropy;
    if (a.stats) {
      a.stats[2 * r] = st.m;
      a.stats[2 * r + 1] = st.log_s;
    }
  }
  // one scan per alternative: the largest (value, lowest index) key below the last one taken
  unsigned long long last = ~0ull;
  auto kmax = [](unsigned long long x, unsigned long long y) { return x > y ? x : y; };
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < a.V; i += NT) {
      const unsigned long long key = ((unsigned long long)order_key(ldf(row + i)) << 32) | (uint32_t)~i;
      if ((k == 0 || key < last) && key > best) best = key;
    }
    last = block_reduce(best, redk, kmax);
    if (threadIdx.x == 0) {
      const int i = (int)~(uint32_t)last;
      a.top_ids[r * a.top_k + k] = i;
      a.top_logprobs[r * a.top_k + k] = log_prob(ldf(row + i), st.m, st.log_s, a.inv_t);
    }
  }
}

struct BwdArgs {
  const int64_t *targets;
  const float *stats, *entropy, *d_logprob, *d_entropy;
  float inv_t;
  int V;
};

// dx_j = (g (1{j = t} - p_j) - h p_j (log p_j + H)) / T
template <typename T>
__global__ void __launch_bounds__(NT) token_logprobs_bwd_kernel(const T *__restrict__ logits, Rows rows, BwdArgs a,
                                                                T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  const int64_t r = blockIdx.x;
  const T *row = logits + rows.at(r);
  T *out = grad + grows.at(r);
  const float m = a.stats[2 * r], log_s = a.stats[2 * r + 1];
  const float h = a.d_entropy ? a.d_entropy[r] : 0.f;
  int64_t t = -1;
  float g = 0.f;
  if (a.d_logprob) {
    t = a.targets[r];
    g = t < 0 ? 0.f : t >= a.V ? NAN : a.d_logprob[r];
  }
  const float ent = a.entropy ? a.entropy[r] : 0.f;
  const bool none = (g == 0.f && h == 0.f) || m == -INFINITY;
  for (int i = threadIdx.x; i < a.V; i += NT) {
    float v = 0.f;
    if (!none) {
      const float lp = (ldf(row + i) - m) * a.inv_t - log_s;
      const float p = expf(lp);
      v = -p * (g + h * (fmaxf(lp, -1000.f) + ent));
      if (i == t) v += g;
      v *= a.inv_t;
    }
    stf(out + i, v);
  }
}

struct DistillArgs {
  const int64_t *ids;
  const void *values;
  int v_dtype, k;
  const float *row_weight;
  float *loss, *stats;
  const float *stats_in;
  float inv_t;
  int V;
};

__device__ __forceinline__ float load_value(const void *p, int64_t i, int dtype) {
  return dtype == MTP_F32    ? ((const float *)p)[i]
         : dtype == MTP_BF16 ? __bfloat162float(((const __nv_bfloat16 *)p)[i])
                             : __half2float(((const __half *)p)[i]);
}

// loss = sum q_i (log q_i - log p_id_i), dx_j = w (sum q p_j - sum_{id_i = j} q_i) / T; q: softmax over the used
// entries of the teacher's logits / T.  GRAD: the gradient is written too.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(NT) distill_kernel(const T *__restrict__ logits, Rows rows, DistillArgs a,
                                                     T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ float red[NT / 32];
  __shared__ int64_t sid[MAX_TOP];
  __shared__ float sq[MAX_TOP];
  const int64_t r = blockIdx.x;
  const T *row = logits + rows.at(r);
  auto fmx = [](float x, float y) { return nan_max(x, y); };
  auto add = [](float x, float y) { return sum_op(x, y); };
  // teacher: thread i holds entry i
  float tv = -INFINITY;
  int64_t id = -1;
  if (threadIdx.x < (unsigned)a.k) {
    id = a.ids[r * a.k + threadIdx.x];
    if (id >= 0) tv = load_value(a.values, r * a.k + threadIdx.x, a.v_dtype);
  }
  const float tm = block_reduce(tv, red, fmx);
  const float td = (tv - tm) * a.inv_t;
  const float te = tv == -INFINITY ? 0.f : expf(td);
  const float ts = block_reduce(te, red, add);
  const bool used = ts != 0.f;
  const float q = used ? te / ts : 0.f;
  const bool bad = q != 0.f && id >= a.V;
  const RowStats st = a.stats_in ? RowStats{a.stats_in[2 * r], a.stats_in[2 * r + 1], 0.f}
                                 : row_stats(row, a.V, a.inv_t, red);
  float term = 0.f;
  if (bad) term = NAN;
  else if (q != 0.f) term = q * ((td - logf(ts)) - log_prob(ldf(row + id), st.m, st.log_s, a.inv_t));
  const float loss = block_reduce(term, red, add);
  if (threadIdx.x == 0) {
    if (a.loss) a.loss[r] = loss;
    if (a.stats) {
      a.stats[2 * r] = st.m;
      a.stats[2 * r + 1] = st.log_s;
    }
  }
  if constexpr (GRAD) {
    if (threadIdx.x < (unsigned)a.k) {
      sid[threadIdx.x] = q != 0.f ? id : -1;
      sq[threadIdx.x] = q;
    }
    const bool any_bad = block_reduce(bad ? 1.f : 0.f, red, add) != 0.f;  // also orders sid / sq
    const float w = a.row_weight[r] * a.inv_t;
    const bool none = !used || w == 0.f || st.m == -INFINITY;
    T *out = grad + grows.at(r);
    for (int i = threadIdx.x; i < a.V; i += NT) {
      float v = 0.f;
      if (!none) {
        v = expf((ldf(row + i) - st.m) * a.inv_t - st.log_s);
        float qs = 0.f;
        for (int j = 0; j < a.k; ++j) qs += sid[j] == i ? sq[j] : 0.f;
        v = any_bad ? NAN : w * (v - qs);
      }
      stf(out + i, v);
    }
  }
}

#define MTP_DISPATCH_LOGITS(code, T, ...)                                    \
  do {                                                                       \
    if ((code) == MTP_F32) { using T = float; __VA_ARGS__; }                 \
    else if ((code) == MTP_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }   \
    else if ((code) == MTP_F16) { using T = __half; __VA_ARGS__; }           \
    else return ::mtp::fail(MTP_ERR_UNSUPPORTED, std::string(__func__) + ": dtype must be F32, BF16 or F16"); \
  } while (0)

#define MTP_REQUIRE_ROWS()                                                                                        \
  MTP_REQUIRE(outer >= 0 && inner >= 0 && ld_outer >= 0 && ld >= 0, "bad sizes");                                 \
  MTP_REQUIRE(V > 0 && V <= (1 << 30), "the vocabulary must have 1 to 2^30 tokens");                              \
  MTP_REQUIRE(inner == 0 || outer <= 0x7fffffffll / inner, "more than 2^31 - 1 rows");                            \
  MTP_REQUIRE(temperature > 0.f && temperature < INFINITY, "temperature must be positive and finite");            \
  if (outer == 0 || inner == 0) return MTP_OK;                                                                    \
  MTP_REQUIRE(logits, "null pointer")

}  // namespace
}  // namespace mtp

using namespace mtp;

extern "C" {

int mtp_token_logprobs(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld, int V,
                       const int64_t *targets, float temperature, float *logprob, float *entropy, float *stats,
                       int top_k, int64_t *top_ids, float *top_logprobs, void *stream) {
  MTP_REQUIRE_ROWS();
  MTP_REQUIRE(!logprob || targets, "logprob needs targets");
  MTP_REQUIRE(top_k >= 0 && top_k <= MAX_TOP && top_k <= V, "top_k must be between 0 and min(V, 128)");
  MTP_REQUIRE(top_k == 0 || (top_ids && top_logprobs), "top_k needs top_ids and top_logprobs");
  cudaStream_t s = (cudaStream_t)stream;
  const Rows rows{inner, ld_outer, ld};
  const FwdArgs a{targets, logprob, entropy, stats, top_k, top_ids, top_logprobs, 1.f / temperature, V};
  MTP_DISPATCH_LOGITS(dtype, T, launch_pdl(token_logprobs_kernel<T>, dim3((unsigned)(outer * inner)), dim3(NT), 0, s,
                                           (const T *)logits, rows, a));
  return check_launch("token_logprobs");
}

int mtp_token_logprobs_bwd(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld,
                           int V, const int64_t *targets, float temperature, const float *stats, const float *entropy,
                           const float *d_logprob, const float *d_entropy, void *grad, int64_t grad_ld_outer,
                           int64_t grad_ld, void *stream) {
  MTP_REQUIRE_ROWS();
  MTP_REQUIRE(stats && grad && grad_ld >= V && grad_ld_outer >= 0, "bad arguments");
  MTP_REQUIRE(!d_logprob || targets, "d_logprob needs targets");
  MTP_REQUIRE(!d_entropy || entropy, "d_entropy needs entropy");
  cudaStream_t s = (cudaStream_t)stream;
  const Rows rows{inner, ld_outer, ld}, grows{inner, grad_ld_outer, grad_ld};
  const BwdArgs a{targets, stats, entropy, d_logprob, d_entropy, 1.f / temperature, V};
  MTP_DISPATCH_LOGITS(dtype, T, launch_pdl(token_logprobs_bwd_kernel<T>, dim3((unsigned)(outer * inner)), dim3(NT), 0, s,
                                           (const T *)logits, rows, a, (T *)grad, grows));
  return check_launch("token_logprobs_bwd");
}

int mtp_distill_topk(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld, int V,
                     const int64_t *ids, const void *values, int v_dtype, int k, float temperature, float *loss,
                     float *stats, void *stream) {
  MTP_REQUIRE_ROWS();
  MTP_REQUIRE(ids && values && loss, "null pointer");
  MTP_REQUIRE(k > 0 && k <= MAX_TOP, "k must be between 1 and 128");
  MTP_REQUIRE(v_dtype == MTP_F32 || v_dtype == MTP_BF16 || v_dtype == MTP_F16, "values must be F32, BF16 or F16");
  cudaStream_t s = (cudaStream_t)stream;
  const Rows rows{inner, ld_outer, ld};
  const DistillArgs a{ids, values, v_dtype, k, nullptr, loss, stats, nullptr, 1.f / temperature, V};
  MTP_DISPATCH_LOGITS(dtype, T, launch_pdl(distill_kernel<T, false>, dim3((unsigned)(outer * inner)), dim3(NT), 0, s,
                                           (const T *)logits, rows, a, (T *)nullptr, rows));
  return check_launch("distill_topk");
}

int mtp_distill_topk_grad(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld,
                          int V, const int64_t *ids, const void *values, int v_dtype, int k, float temperature,
                          const float *stats, const float *row_weight, float *loss, void *grad, int64_t grad_ld_outer,
                          int64_t grad_ld, void *stream) {
  MTP_REQUIRE_ROWS();
  MTP_REQUIRE(ids && values && row_weight && grad && grad_ld >= V && grad_ld_outer >= 0, "bad arguments");
  MTP_REQUIRE(k > 0 && k <= MAX_TOP, "k must be between 1 and 128");
  MTP_REQUIRE(v_dtype == MTP_F32 || v_dtype == MTP_BF16 || v_dtype == MTP_F16, "values must be F32, BF16 or F16");
  cudaStream_t s = (cudaStream_t)stream;
  const Rows rows{inner, ld_outer, ld}, grows{inner, grad_ld_outer, grad_ld};
  const DistillArgs a{ids, values, v_dtype, k, row_weight, loss, nullptr, stats, 1.f / temperature, V};
  MTP_DISPATCH_LOGITS(dtype, T, launch_pdl(distill_kernel<T, true>, dim3((unsigned)(outer * inner)), dim3(NT), 0, s,
                                           (const T *)logits, rows, a, (T *)grad, grows));
  return check_launch("distill_topk_grad");
}

// Rows of fp32 logits that one pass of mtp_lm_head_logprobs holds: about 256 MB of them.
static int64_t score_block(int64_t rows, int V) {
  int64_t b = (256ll << 20) / (4ll * V);
  b = b < 128 ? 128 : b / 128 * 128;
  return rows < b ? rows : b;
}
static int64_t score_ld(int V) { return ((int64_t)V + 7) / 8 * 8; }

int mtp_lm_head_logprobs_workspace(int rows, int V, int K, int dtype, int top_k, int64_t *bytes) {
  MTP_REQUIRE(rows >= 0 && V > 0 && V <= (1 << 30) && K > 0 && top_k >= 0 && bytes, "bad arguments");
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16, "dtype must be F32 or BF16");
  *bytes = score_block(rows, V) * score_ld(V) * 4;
  return MTP_OK;
}

int mtp_lm_head_logprobs(const void *hidden, int ld_hidden, int rows, int K, const void *weight, int ld_weight, int V,
                         int dtype, const int64_t *targets, float temperature, float *logprob, float *entropy,
                         int top_k, int64_t *top_ids, float *top_logprobs, void *workspace, int64_t workspace_bytes,
                         void *stream) {
  MTP_REQUIRE(rows >= 0 && V > 0 && V <= (1 << 30) && K > 0 && ld_hidden >= K && ld_weight >= K, "bad sizes");
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16, "dtype must be F32 or BF16");
  MTP_REQUIRE(temperature > 0.f && temperature < INFINITY, "temperature must be positive and finite");
  MTP_REQUIRE(top_k >= 0 && top_k <= MAX_TOP && top_k <= V, "top_k must be between 0 and min(V, 128)");
  if (rows == 0) return MTP_OK;
  MTP_REQUIRE(hidden && weight && workspace, "null pointer");
  MTP_REQUIRE(!logprob || targets, "logprob needs targets");
  MTP_REQUIRE(top_k == 0 || (top_ids && top_logprobs), "top_k needs top_ids and top_logprobs");
  int64_t need = 0;
  mtp_lm_head_logprobs_workspace(rows, V, K, dtype, top_k, &need);
  MTP_REQUIRE(workspace_bytes >= need && aligned16(workspace), "workspace too small or not 16-byte aligned");
  const int64_t blk = score_block(rows, V), ld = score_ld(V);
  const size_t es = dtype == MTP_F32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < rows; r0 += blk) {
    const int n = (int)(rows - r0 < blk ? rows - r0 : blk);
    int rc = mtp_gemm((const char *)hidden + (size_t)r0 * ld_hidden * es, weight, workspace, n, V, K, ld_hidden, ld_weight,
                      (int)ld, dtype, MTP_F32, MTP_EPI_STORE, nullptr, 0, stream);
    if (rc) return rc;
    rc = mtp_token_logprobs(workspace, MTP_F32, 1, n, 0, ld, V, targets ? targets + r0 : nullptr, temperature,
                            logprob ? logprob + r0 : nullptr, entropy ? entropy + r0 : nullptr, nullptr, top_k,
                            top_ids ? top_ids + r0 * top_k : nullptr, top_logprobs ? top_logprobs + r0 * top_k : nullptr,
                            stream);
    if (rc) return rc;
  }
  return MTP_OK;
}

}  // extern "C"

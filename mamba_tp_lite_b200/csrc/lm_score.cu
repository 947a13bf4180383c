// Log probabilities straight from hidden states: x = hidden[M, K] . weight[V, K]^T with the softmax statistics of every
// row in the GEMM's epilogue; the logits stay in tensor memory and are never written.
//
// Persistent, warp-specialised CTA (one per SM), tiles of 128 rows x bn tokens:
//   warp 0     one lane issues TMA tile loads (hidden 128x64, weight bn x 64, 128-byte swizzle) into a 4-stage ring;
//   warp 1     allocates 512 TMEM columns (two 128 x bn fp32 accumulators), one lane issues tcgen05.mma;
//   warps 2-9  epilogue: two warps per TMEM lane quarter, each on half of the tile's columns, a lane holding one row.
//              A lane adds the accumulators of the splits of K in registers, then keeps the running (m, S, U) of its
//              columns; the second warp hands its own to the first through shared memory, and one (m, S, U) per row and
//              tile goes to the workspace, the given token's logit beside it.
// A second kernel joins a row's tiles.  K is split because the tensor core truncates at every step of its sum: measured
// against 64 bits, a sum over K is 8.6e-10 K of its value too small (1.8e-6 at K = 2048, which an entropy shows).  Every
// further split costs a tile 300 to 900 cycles, in which the accumulator is read (8192 rows of K = 2048, V = 50280: 1107 us
// unsplit, 1124 with two splits, 1186 with four, 1384 with eight), so that one sums up to 1024.
// The epilogue works on a tile while the tensor core fills the next one's accumulators.
// Every mbarrier wait is bounded; a CTA that gives up marks its status slot, frees its TMEM and returns, and the second
// kernel then writes NaN.
#include <type_traits>
#include "common.cuh"
#include "logits.cuh"
#include "tc_common.cuh"

namespace mtp {
bool gemm_tc_eligible(const void *A, const void *B, int M, int N, int K, int lda, int ldb);
bool gemm_on_tensor_cores(const void *A, const void *B, int M, int N, int K, int lda, int ldb, int ab_dtype);
int gemm_tc(const void *A, const void *B, void *C, int M, int N, int K, int lda, int ldb, int ldc, int c_dtype, int epi,
            const void *bias, int bias_dtype, cudaStream_t stream, int *expired);
int launch_token_logprobs(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld, int V,
                          const int64_t *targets, float temperature, float *logprob, float *entropy, float *stats, int top_k,
                          int64_t *top_ids, float *top_logprobs, const int *expired, cudaStream_t stream);

namespace {

using namespace lg;
using namespace tc;

constexpr int BM = 128, BK = 64, BN_MAX = 256, STAGES = 4;
constexpr int SPLIT = 16;  // K blocks that one accumulator sums, at most
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN_MAX * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int EPI_WARPS = 8, NUM_THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 512;
constexpr int HAND_BYTES = 2 * 4 * 32 * 12;  // [tile parity][lane quarter][lane] (m, S, U)
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align slack*/ + 256 /*barriers*/ + HAND_BYTES;
constexpr unsigned long long TIMEOUT_NS = 2000000000ull;

struct ScoreParams {
  const int64_t *targets;
  float *part;    // [3][tiles_n][M]: m, S, U
  float *hit;     // [M] the given token's logit
  int *status;    // [gridDim.x]
  int M, N, K;
  int bn, tiles_m, tiles_n, num_tiles, group_m;
  int a_rows;  // rows of a hidden-state box
  int split;   // K blocks that one accumulator sums
  uint32_t idesc;
  float c2;
};

// Tiles in groups of group_m row blocks, rows fastest: the CTAs at work share weight tiles, and the group's hidden states
// (32 x 128 x K) stay in L2.
__device__ __forceinline__ void tile_coords(const ScoreParams &p, int t, int &mt, int &nt) {
  const int gsize = p.group_m * p.tiles_n;
  const int g = t / gsize;
  const int first_m = g * p.group_m;
  const int gm = min(p.tiles_m - first_m, p.group_m);
  const int r = t - g * gsize;
  mt = first_m + r % gm;
  nt = r / gm;
}

// h = v where at == i.  (Written out, so that a row of them is not turned into an indexed array in local memory.)
__device__ __forceinline__ void pick(float &h, float v, int at, int i) {
  asm("{\n.reg .pred p;\nsetp.eq.s32 p, %2, %3;\nselp.f32 %0, %1, %0, p;\n}" : "+f"(h) : "f"(v), "r"(at), "r"(i));
}

template <bool ENT>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    lm_score_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const ScoreParams p) {
  extern __shared__ __align__(1024) unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char *gbase = smem_dyn + (base - raw);
  const uint32_t bar0 = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 4);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(gbase + STAGES * STAGE_BYTES + 8 * (2 * STAGES + 5));
  volatile int *abort = reinterpret_cast<volatile int *>(gbase + STAGES * STAGE_BYTES + 8 * (2 * STAGES + 5) + 8);
  float *hand = reinterpret_cast<float *>(gbase + STAGES * STAGE_BYTES + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  MTP_PDL_WAIT();  // barrier init and TMEM allocation above overlap the previous kernel
  MTP_PDL_TRIGGER();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = (p.K + BK - 1) / BK;
  const uint32_t tx_bytes = (uint32_t)((p.a_rows + p.bn) * BK * 2);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      for (int t = blockIdx.x; t < p.num_tiles && !*abort; t += gridDim.x) {
        int mt, nt;
        tile_coords(p, t, mt, nt);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort, TIMEOUT_NS)) break;
          mbar_expect_tx(full_bar(s), tx_bytes);
          const uint32_t sa = base + s * STAGE_BYTES;
          tma_load_2d(sa, &tmA, full_bar(s), kb * BK, mt * BM);
          tma_load_2d(sa + A_BYTES, &tmB, full_bar(s), kb * BK, nt * p.bn);
          ++issued;
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
      if (*abort) {  // wait (bounded) until the most recent fills have landed
        const int back = issued < STAGES ? issued : STAGES;
        for (int i = 0; i < back; ++i) {
          if (--s < 0) { s = STAGES - 1; ph ^= 1u; }
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(full_bar(s), ph) && globaltimer_ns() - t0 < 100000000ull) {}
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int s = 0, local = 0;
      uint32_t ph = 0;
      bool any = false;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < p.num_tiles && !*abort; t += gridDim.x) {
        for (int kb0 = 0; ok && kb0 < num_kb; kb0 += p.split, ++local) {
          const int a = local & 1;
          const uint32_t use = (uint32_t)(local >> 1);
          if (!mbar_wait(tempty_bar(a), (use & 1u) ^ 1u, abort, TIMEOUT_NS)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)(a * BN_MAX);
          const int nkb = min(p.split, num_kb - kb0);
          for (int kb = 0; kb < nkb; ++kb) {
            if (!mbar_wait(full_bar(s), ph, abort, TIMEOUT_NS)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sa = base + s * STAGE_BYTES;
            const uint64_t ad = sw128_desc(sa), bd = sw128_desc(sa + A_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)  // +32 bytes along K per instruction
              umma_bf16(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), p.idesc, (kb | k) != 0);
            any = true;
            umma_commit(empty_bar(s));
            if (++s == STAGES) { s = 0; ph ^= 1u; }
          }
          if (ok) umma_commit(tfull_bar(a));
        }
      }
      if (*abort && any) {
        umma_commit(drain_bar);
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(drain_bar, 0) && globaltimer_ns() - t0 < 100000000ull) {}
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const int q = warp & 3;           // TMEM lane quarter this warp may access
    const int half = (warp - 2) >> 2;  // its half of the tile's 16-column chunks
    const int chunks = p.bn / 16, cut = (chunks + 1) / 2;
    const int c_lo = half ? cut : 0, c_hi = half ? chunks : cut;
    const int nch = c_hi - c_lo;
    int local = 0, tile = 0;
    bool alive = true;
    for (int t = blockIdx.x; t < p.num_tiles; t += gridDim.x, ++tile) {
      int mt, nt;
      tile_coords(p, t, mt, nt);
      const int row = mt * BM + q * 32 + lane;
      int64_t tgt = -1;
      if (p.targets && row < p.M) tgt = p.targets[row];
      const int64_t rel = tgt - (int64_t)nt * p.bn;  // the given token's column of this tile, if it is in it
      const int at = rel >= 0 && rel < p.bn && tgt < p.N ? (int)rel : -16;
      F2 acc[BN_MAX / 32][8];  // this lane's sums so far: half a tile
      Stat st{LOWEST, 0.f, 0.f};
      auto chunk = [&](int c, const F2 (&x)[8]) {
        const int n0 = nt * p.bn + 16 * (c_lo + c);
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) un2(x[i], v[2 * i], v[2 * i + 1]);
        if (n0 + 16 > p.N) {  // tokens past the vocabulary
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (n0 + i >= p.N) v[i] = -INFINITY;
        }
        if ((at >> 4) == c_lo + c) {
          float h = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) pick(h, v[i], at & 15, i);
          p.hit[row] = h;
        }
        bool masked;
        accumulate<ENT, 16>(st, v, p.c2, masked);
      };
      for (int kb0 = 0; kb0 < num_kb; kb0 += p.split, ++local) {
        const int a = local & 1;
        const uint32_t use = (uint32_t)(local >> 1);
        // a warp that gives up still meets its partner at the barrier below
        alive = __all_sync(0xffffffffu, alive && mbar_wait(tfull_bar(a), use & 1u, abort, TIMEOUT_NS));
        tc_fence_after();
        if (alive) {
          const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * BN_MAX + 16 * c_lo);
          auto take = [&](auto first) {
#pragma unroll
            for (int c = 0; c < BN_MAX / 32; ++c) {
              if (c < nch) {
                float v[16];
                tmem_ld16(tbase + 16u * c, v);
                F2 x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  x[i] = f2(v[2 * i], v[2 * i + 1]);
                  acc[c][i] = first ? x[i] : add2(acc[c][i], x[i]);
                }
              }
            }
          };
          if (kb0 == 0) take(std::true_type{});
          else take(std::false_type{});
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(a));
      }
      if (alive) {
#pragma unroll
        for (int c = 0; c < BN_MAX / 32; ++c)
          if (c < nch) chunk(c, acc[c]);
      }
      // the second half's statistics to the first; the buffer alternates by tile, so one barrier a tile orders both uses
      float *h = hand + (((tile & 1) * 4 + q) * 32 + lane) * 3;
      if (half) {
        h[0] = st.m;
        h[1] = st.s;
        h[2] = st.u;
      }
      asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
      if (!half && row < p.M) {
        st = join<ENT>(st, Stat{h[0], h[1], h[2]}, p.c2);
        const int64_t at_part = (int64_t)nt * p.M + row, plane = (int64_t)p.tiles_n * p.M;
        p.part[at_part] = st.m;
        p.part[plane + at_part] = st.s;
        if (ENT) p.part[2 * plane + at_part] = st.u;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) p.status[blockIdx.x] = *abort;
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
}

// Joins the tiles of a row: 8 rows per CTA, 32 threads a row (4 lanes of each warp, so that a warp reads four 32-byte
// sectors), eight tiles in flight per thread: one round of loads up to 256 tiles.
constexpr int JOIN_WARPS = 8, JOIN_ROWS = 8;
template <bool ENT>
__global__ void __launch_bounds__(32 * JOIN_WARPS) lm_score_join_kernel(const ScoreParams p, int ctas, float inv_t,
                                                                        float *__restrict__ logprob,
                                                                        float *__restrict__ entropy) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  constexpr int STRIDE = 4 * JOIN_WARPS;
  __shared__ Stat sh[JOIN_WARPS][JOIN_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * JOIN_ROWS + (lane & 7);
  int gave_up = 0;
  for (int i = threadIdx.x; i < ctas; i += 32 * JOIN_WARPS) gave_up |= p.status[i];
  Stat st{LOWEST, 0.f, 0.f};
  if (row < p.M) {
    const int64_t plane = (int64_t)p.tiles_n * p.M;
    for (int t = warp * 4 + (lane >> 3); t < p.tiles_n; t += 8 * STRIDE) {
      Stat s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tj = t + j * STRIDE;
        s[j] = Stat{LOWEST, 0.f, 0.f};
        if (tj < p.tiles_n) {
          const int64_t at = (int64_t)tj * p.M + row;
          s[j] = Stat{p.part[at], p.part[plane + at], ENT ? p.part[2 * plane + at] : 0.f};
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) st = join<ENT>(st, s[j], p.c2);
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o *= 2) {
    Stat other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.u = ENT ? __shfl_xor_sync(0xffffffffu, st.u, o) : 0.f;
    st = join<ENT>(st, other, p.c2);
  }
  if (lane < JOIN_ROWS) sh[warp][lane] = st;
  gave_up = __syncthreads_or(gave_up);
  if (threadIdx.x >= JOIN_ROWS || row >= p.M) return;
  for (int w = 1; w < JOIN_WARPS; ++w) st = join<ENT>(st, sh[w][lane], p.c2);
  const RowStats r = gave_up ? expired() : finish(st);
  if (logprob) {
    const int64_t t = p.targets[row];
    logprob[row] = t < 0 ? 0.f : t >= p.N ? NAN : log_prob(p.hit[row], r.m, r.log_s, inv_t);
  }
  if (entropy) entropy[row] = r.entropy;
}

struct ScorePlan {
  int bn, tiles_m, tiles_n, grid;
  int64_t hit, status, bytes;  // offsets into the workspace, and its size
};

// Tile width: the multiple of 16 up to 256 that gives the shortest longest CTA, a tile costing its width and 48 columns'
// time on top.  Measured at V = 50280, both kernels, L2 cold: 64 rows, K = 768 (one row block) 32.0 us at the chosen 176
// against 34.8 at 256; 8192 rows, K = 2048 1124 us at the chosen 256 against 1138 at 240 and 1290 at 192.
ScorePlan score_plan(int rows, int V) {
  ScorePlan p;
  const int sms = num_sms();
  p.tiles_m = ceil_div(rows, BM);
  long best = -1;
  for (int bn = BN_MAX; bn >= 32; bn -= 16) {
    const long tiles = (long)p.tiles_m * ceil_div(V, bn);
    const long cost = (tiles + sms - 1) / sms * (bn + 48);
    if (best < 0 || cost < best) {
      best = cost;
      p.bn = bn;
    }
  }
  p.tiles_n = ceil_div(V, p.bn);
  const long tiles = (long)p.tiles_m * p.tiles_n;
  p.grid = (int)(tiles < sms ? tiles : sms);
  p.hit = 12ll * p.tiles_n * rows;
  p.status = p.hit + 4ll * rows;
  p.bytes = p.status + 4ll * p.grid;
  return p;
}

// Rows of fp32 logits that one pass of the unfused form holds: about 256 MB of them, and no more than the grid of the
// CUDA-core product has places for (65535 tiles of 64 rows).
int64_t score_ld(int V) { return ((int64_t)V + 7) / 8 * 8; }
int64_t score_block(int64_t rows, int V) {
  int64_t b = (256ll << 20) / (4 * score_ld(V)) / 128 * 128;
  b = b < 128 ? 128 : b > 65535 / 2 * 128 ? 65535 / 2 * 128 : b;
  return rows < b ? rows : b;
}
// Behind them 16 bytes for a word that says whether a wait of one of the products has expired.
int64_t score_block_bytes(int64_t rows, int V) { return score_block(rows, V) * score_ld(V) * 4; }

// The fused kernel takes bf16 operands that TMA can read, and gives no alternatives.
bool score_fused(const void *hidden, int ld_hidden, int rows, int K, const void *weight, int ld_weight, int V, int dtype,
                 int top_k) {
  return dtype == MTP_BF16 && top_k == 0 && gemm_tc_eligible(hidden, weight, rows, V, K, ld_hidden, ld_weight) &&
         (int64_t)ceil_div(rows, BM) * ceil_div(V, 32) < 0x7fffffffll;
}

int launch_score(const void *hidden, int ld_hidden, int rows, int K, const void *weight, int ld_weight, int V,
                 const int64_t *targets, float temperature, float *logprob, float *entropy, char *ws, cudaStream_t stream) {
  const ScorePlan plan = score_plan(rows, V);
  ScoreParams p{};
  p.targets = logprob ? targets : nullptr;
  p.part = (float *)ws;
  p.hit = (float *)(ws + plan.hit);
  p.status = (int *)(ws + plan.status);
  p.M = rows;
  p.N = V;
  p.K = K;
  p.bn = plan.bn;
  p.tiles_m = plan.tiles_m;
  p.tiles_n = plan.tiles_n;
  p.num_tiles = plan.tiles_m * plan.tiles_n;
  p.group_m = 32;
  // one row block: only the 8-row groups that hold rows are loaded; the MMA's other rows are whatever the ring held, and
  // their accumulators are not read
  p.a_rows = rows < BM ? (rows + 7) / 8 * 8 : BM;
  const int num_kb = (K + BK - 1) / BK, splits = (num_kb + SPLIT - 1) / SPLIT;
  p.split = (num_kb + splits - 1) / splits;
  p.idesc = idesc_bf16(BM, plan.bn);
  p.c2 = (float)(1.4426950408889634 / temperature);
  CUtensorMap ta, tb;
  int rc = make_tmap(&ta, hidden, rows, K, ld_hidden, p.a_rows);
  if (rc) return rc;
  rc = make_tmap(&tb, weight, V, K, ld_weight, plan.bn);
  if (rc) return rc;
  auto kern = entropy ? lm_score_kernel<true> : lm_score_kernel<false>;
  // set at every call: the attribute belongs to the current device
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) {
    cudaGetLastError();
    return fail(MTP_ERR_CUDA, "lm_score: shared memory");
  }
  launch_pdl(kern, dim3(plan.grid), dim3(NUM_THREADS), SMEM_BYTES, stream, ta, tb, p);
  rc = check_launch("lm_score");
  if (rc) return rc;
  auto join = entropy ? lm_score_join_kernel<true> : lm_score_join_kernel<false>;
  launch_pdl(join, dim3(ceil_div(rows, JOIN_ROWS)), dim3(32 * JOIN_WARPS), 0, stream, p, plan.grid, 1.f / temperature, logprob,
             entropy);
  return check_launch("lm_score_join");
}

}  // namespace
}  // namespace mtp

using namespace mtp;

extern "C" {

int mtp_lm_head_logprobs_workspace(const void *hidden, int ld_hidden, int rows, int K, const void *weight, int ld_weight,
                                   int V, int dtype, int top_k, int64_t *bytes) {
  MTP_REQUIRE(rows >= 0 && V > 0 && V <= (1 << 30) && K > 0 && top_k >= 0 && bytes, "bad arguments");
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16, "dtype must be F32 or BF16");
  if (score_fused(hidden, ld_hidden, rows, K, weight, ld_weight, V, dtype, top_k))
    *bytes = score_plan(rows, V).bytes;
  else
    *bytes = score_block_bytes(rows, V) + 16;
  return MTP_OK;
}

int mtp_lm_head_logprobs(const void *hidden, int ld_hidden, int rows, int K, const void *weight, int ld_weight, int V,
                         int dtype, const int64_t *targets, float temperature, float *logprob, float *entropy,
                         int top_k, int64_t *top_ids, float *top_logprobs, void *workspace, int64_t workspace_bytes,
                         void *stream) {
  MTP_REQUIRE(rows >= 0 && V > 0 && V <= (1 << 30) && K > 0 && ld_hidden >= K && ld_weight >= K, "bad sizes");
  MTP_REQUIRE(dtype == MTP_F32 || dtype == MTP_BF16, "dtype must be F32 or BF16");
  MTP_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "temperature must be between 1e-6 and 1e6");
  MTP_REQUIRE(top_k >= 0 && top_k <= 128 && top_k <= V, "top_k must be between 0 and min(V, 128)");
  if (rows == 0) return MTP_OK;
  MTP_REQUIRE(hidden && weight && workspace, "null pointer");
  MTP_REQUIRE(!logprob || targets, "logprob needs targets");
  MTP_REQUIRE(top_k == 0 || (top_ids && top_logprobs), "top_k needs top_ids and top_logprobs");
  int64_t need = 0;
  mtp_lm_head_logprobs_workspace(hidden, ld_hidden, rows, K, weight, ld_weight, V, dtype, top_k, &need);
  MTP_REQUIRE(workspace_bytes >= need && aligned16(workspace), "workspace too small or not 16-byte aligned");
  if (score_fused(hidden, ld_hidden, rows, K, weight, ld_weight, V, dtype, top_k))
    return launch_score(hidden, ld_hidden, rows, K, weight, ld_weight, V, targets, temperature, logprob, entropy,
                        (char *)workspace, (cudaStream_t)stream);
  const int64_t blk = score_block(rows, V), ld = score_ld(V);
  const size_t es = dtype == MTP_F32 ? 4 : 2;
  cudaStream_t st = (cudaStream_t)stream;
  int *expired = nullptr;
  if (gemm_on_tensor_cores(hidden, weight, rows, V, K, ld_hidden, ld_weight, dtype)) {
    expired = (int *)((char *)workspace + score_block_bytes(rows, V));
    if (cudaMemsetAsync(expired, 0, sizeof(int), st) != cudaSuccess) {
      cudaGetLastError();
      return fail(MTP_ERR_CUDA, "mtp_lm_head_logprobs: could not clear the status word");
    }
  }
  for (int64_t r0 = 0; r0 < rows; r0 += blk) {
    const int n = (int)(rows - r0 < blk ? rows - r0 : blk);
    const char *h = (const char *)hidden + (size_t)r0 * ld_hidden * es;
    int rc = gemm_on_tensor_cores(h, weight, n, V, K, ld_hidden, ld_weight, dtype)
                 ? gemm_tc(h, weight, workspace, n, V, K, ld_hidden, ld_weight, (int)ld, MTP_F32, MTP_EPI_STORE, nullptr, 0,
                           st, expired)
                 : mtp_gemm(h, weight, workspace, n, V, K, ld_hidden, ld_weight, (int)ld, dtype, MTP_F32, MTP_EPI_STORE,
                            nullptr, 0, stream);
    if (rc) return rc;
    rc = launch_token_logprobs(workspace, MTP_F32, 1, n, 0, ld, V, targets ? targets + r0 : nullptr, temperature,
                               logprob ? logprob + r0 : nullptr, entropy ? entropy + r0 : nullptr, nullptr, top_k,
                               top_ids ? top_ids + r0 * top_k : nullptr,
                               top_logprobs ? top_logprobs + r0 * top_k : nullptr, expired, st);
    if (rc) return rc;
  }
  return MTP_OK;
}

}  // extern "C"

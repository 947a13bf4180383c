// The int8 product on the tensor cores: tcgen05.mma kind::i8, int32 accumulators in tensor memory.
//
// Persistent, warp-specialised, one CTA per SM; CG = 2 pairs the CTAs of two SMs on one 256 x bn tile, each with its own 128
// rows of a and half of the tile's rows of w, so that a row of w is loaded once for 256 rows of a:
//   warp 0     one lane issues the TMA loads of its CTA (128-byte wide boxes, 128-byte swizzle) into a ring;
//   warp 1     allocates tensor memory (two accumulators of 128 lanes x 256 columns); in the pair's first CTA one lane issues
//              tcgen05.mma for both, releases ring slots and signals finished accumulators in both CTAs with tcgen05.commit;
//   warps 2-9  epilogue, two warps per lane quarter, each on every second block of 128 bytes of output columns: sums to fp32,
//              times the row's scale (a lane has one row) and the columns' (from shared memory), rounded into a staging block
//              in the swizzled layout of a TMA store.  It works on one tile while the tensor cores fill the other accumulator.
// Bound by the tensor cores and by what feeds them: at full rate the pair's 256 x 256 tile takes 64 bytes a clock and SM from
// L2, all that a port gives; without the products the copies alone take two thirds of the time.  Measured on a B200 (TOP/s;
// nominal 4500, 3360 being twice the measured bf16 rate): 32768 x 2048 -> 8192 bf16 378 us, 2900; 32768 x 4096 -> 2048 172 us,
// 3190; 8192 x 2048 -> 8192 95 us, 2890.  To K = 1024 the epilogue bounds it, 2.6 us for a tile of a pair: 8192 x 1024 ->
// 16384 109 us (3.5 us a tile and 131 with the arrival at the other CTA's barrier as a release of the cluster's scope, which
// waits for all stores of its thread, and with divisions for a tile's coordinates).
// Every wait is bounded.  Where one expires, the CTA gives NaN for what it has left (the split-K form: for all results of its
// cluster), and when all its warps are through waits, again with a limit, for its copies and products in flight, frees its
// tensor memory and returns.
#include "int8_linear.cuh"
#include "tc_common.cuh"

namespace mtp {
namespace i8 {
namespace {

using namespace tc;

constexpr int BM = 128, BK = 128, BN_MAX = 256;  // rows of a per CTA, bytes of K per ring slot, columns per tile
constexpr int EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 512;
constexpr unsigned long long TIMEOUT_NS = 2000000000ull;
constexpr int A_BYTES = BM * BK;
constexpr int CHUNK_BYTES = 32 * 128;  // 32 rows x 128 bytes of output

constexpr int B_BYTES = 128 * BK;  // at most 128 rows of w per CTA: bn = 256 takes a pair
constexpr int SLOT = A_BYTES + B_BYTES, STAGES = 5;
constexpr int STAGE_OUT = STAGES * SLOT;                    // the epilogue's blocks, one per warp
constexpr int COLS = STAGE_OUT + EPI_WARPS * CHUNK_BYTES;   // scales and biases of a warp's columns
constexpr int BARS = COLS + EPI_WARPS * BN_MAX * 4;
constexpr int SMEM_BYTES = BARS + 256 + 1024 /* to align the base */;

struct Params {
  Out o;
  int M, N, K;
  int bn, tiles_m, tiles_n, num_tiles, group_m;
  int tma_cols;  // blocks of results that end by this column go by TMA stores
  uint32_t idesc;
  unsigned long long timeout_ns;
  uint64_t div_group, div_m, div_last;  // 2^64 / n, rounded up, for a group's tiles, its rows and the last group's rows
};

// Tiles in groups of group_m rows of tiles, rows fastest.  Divisions by multiplication: three by the instruction's way took a
// tile's epilogue 600 cycles.
__device__ __forceinline__ int div_by(int n, uint64_t m) { return (int)__umul64hi((uint64_t)(uint32_t)n, m); }
__device__ __forceinline__ void tile_coords(const Params &p, int t, int &mt, int &nt) {
  const int g = div_by(t, p.div_group), r = t - g * p.group_m * p.tiles_n;
  const int first_m = g * p.group_m, gm = min(p.tiles_m - first_m, p.group_m);
  nt = gm == 1 ? r : div_by(r, gm == p.group_m ? p.div_m : p.div_last);
  mt = first_m + r - nt * gm;
}

__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y) {
  if (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(tm), "r"(bar), "r"(x), "r"(y)
                 : "memory");
  else
    tma_load_2d(dst, tm, bar, x, y);
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// Arrives at `bar` (of both CTAs of a pair) when the products issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    umma_commit(bar);
}

// 32 columns of a warp's lane quarter; tcgen05.wait::ld comes before they are used.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// After an expired wait, by the thread that has issued them: until the last fills of a ring have landed (100 ms at most), s being
// the slot that would be next and ph its parity.
template <typename Bar>
__device__ __forceinline__ void drain_fills(Bar full_bar, int slots, int issued, int s, uint32_t ph) {
  const unsigned long long t0 = globaltimer_ns();
  for (int i = 0; i < issued && i < slots; ++i) {
    if (--s < 0) { s = slots - 1; ph ^= 1u; }
    while (!mbar_try_wait(full_bar(s), ph) && globaltimer_ns() - t0 < 100000000ull) {}
  }
}
// The same for the products that a commit to `bar` (its first phase) follows.
__device__ __forceinline__ void drain_products(uint32_t bar) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, 0) && globaltimer_ns() - t0 < 100000000ull) {}
}

template <typename T> constexpr int PER_WORD = 16 / (int)sizeof(T);  // results in 16 bytes

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <int CG, typename T>
__global__ void __launch_bounds__(THREADS, 1)
    int8_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmC, const Params p) {
  extern __shared__ __align__(1024) unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;  // the same in both CTAs of a pair
  unsigned char *gbase = smem_dyn + (base - raw);
  const uint32_t bar0 = base + BARS;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 4);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(gbase + BARS + 8 * (2 * STAGES + 5));
  volatile int *abort = reinterpret_cast<volatile int *>(gbase + BARS + 8 * (2 * STAGES + 5) + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank = 0;
  if (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), EPI_WARPS * CG);
    }
    mbar_init(drain_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(TMEM_COLS));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // both CTAs' barriers are ready
  tc_fence_after();
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = (p.K + BK - 1) / BK;
  const int b_rows = p.bn / CG;
  // of the threads that issue copies and products: the ring's next slot, its parity, and how many (whether any) were issued
  int s = 0, issued = 0;
  uint32_t ph = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      const uint32_t tx_bytes = (uint32_t)((BM + b_rows) * BK * CG);
      for (int t = first; t < p.num_tiles && !*abort; t += step) {
        int mt, nt;
        tile_coords(p, t, mt, nt);
        const int y_a = (mt * CG + (int)rank) * BM, y_b = nt * p.bn + (int)rank * b_rows;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, abort, p.timeout_ns)) break;
          if (rank == 0) mbar_expect_tx(full_bar(s), tx_bytes);  // both CTAs' bytes count at the first's barrier
          const uint32_t bar = CG == 2 ? cluster_addr(full_bar(s), 0) : full_bar(s);
          const uint32_t sa = base + s * SLOT;
          load_box<CG>(sa, &tmA, bar, kb * BK, y_a);
          load_box<CG>(sa + A_BYTES, &tmB, bar, kb * BK, y_b);
          ++issued;
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0) {
      int local = 0;
      bool ok = true;
      for (int t = first; ok && t < p.num_tiles && !*abort; t += step, ++local) {
        const int a = local & 1;
        const uint32_t use = (uint32_t)(local >> 1);
        if (!mbar_wait(tempty_bar(a), (use & 1u) ^ 1u, abort, p.timeout_ns)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(a * BN_MAX);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(full_bar(s), ph, abort, p.timeout_ns)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = base + s * SLOT;
          const uint64_t ad = sw128_desc(sa), bd = sw128_desc(sa + A_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)  // 32 bytes along K per instruction; past K both operands are zeros
            mma<CG>(d, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), p.idesc, (kb | k) != 0);
          issued = 1;
          commit<CG>(empty_bar(s));
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
        if (ok) commit<CG>(tfull_bar(a));
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    constexpr int CW = 128 / (int)sizeof(T);  // columns of a block of output
    const int q = warp & 3, half = (warp - 2) >> 2;
    unsigned char *stage = gbase + STAGE_OUT + (warp - 2) * CHUNK_BYTES;
    // this warp's columns of a tile, block after block: their scales, and after 128 of them their biases
    float *sw = reinterpret_cast<float *>(gbase + COLS) + (warp - 2) * 256, *sb = sw + 128;
    constexpr int HELD = 128 / 32;  // of them, a lane's
    int local = 0;
    bool alive = true;
    // fetched one tile ahead: the scale of this lane's row, and of its columns
    float next_a = 0.f, next_w[HELD] = {}, next_b[HELD] = {};
    auto fetch = [&](int t) {
      if (t >= p.num_tiles) return;
      int mt, nt;
      tile_coords(p, t, mt, nt);
      const int m = (mt * CG + (int)rank) * BM + q * 32 + lane;
      next_a = m < p.M ? p.o.a_scale[m] : 0.f;
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int i = 32 * j + lane, c = (i / CW * 2 + half) * CW + i % CW, n = nt * p.bn + c;
        const bool in = c < p.bn && n < p.N;
        next_w[j] = in ? p.o.w_scale[n] : 0.f;
        next_b[j] = in ? ld_bias(p.o, n) : 0.f;
      }
    };
    fetch(first);
    for (int t = first; t < p.num_tiles; t += step, ++local) {
      int mt, nt;
      tile_coords(p, t, mt, nt);
      const int a = local & 1;
      const uint32_t use = (uint32_t)(local >> 1);
      const int n_tile = nt * p.bn, m0 = (mt * CG + (int)rank) * BM + q * 32;
      const float sa = next_a;
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        sw[32 * j + lane] = next_w[j];
        sb[32 * j + lane] = next_b[j];
      }
      __syncwarp();
      fetch(t + step);
      alive = __all_sync(0xffffffffu, alive && mbar_wait(tfull_bar(a), use & 1u, abort, p.timeout_ns));
      tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * BN_MAX);
      int at_col = 0;
      for (int c0 = half * CW; c0 < p.bn; c0 += 2 * CW, at_col += CW) {
        if (n_tile + c0 >= p.N || m0 >= p.M) break;
        int acc[CW] = {};
        if (alive) {
#pragma unroll
          for (int g = 0; g < CW; g += 32) tmem_ld32(tbase + (uint32_t)(c0 + g), acc + g);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        uint4 word[8];  // 128 bytes of this lane's row
        constexpr int PER = PER_WORD<T>;
#pragma unroll
        for (int i = 0; i < CW; i += PER) {
          float v[PER];
#pragma unroll
          for (int k = 0; k < PER; k += 4) {
            const float4 w4 = *reinterpret_cast<const float4 *>(sw + at_col + i + k);
            v[k] = scaled(acc[i + k], sa, w4.x);
            v[k + 1] = scaled(acc[i + k + 1], sa, w4.y);
            v[k + 2] = scaled(acc[i + k + 2], sa, w4.z);
            v[k + 3] = scaled(acc[i + k + 3], sa, w4.w);
            if (p.o.bias) {
              const float4 b4 = *reinterpret_cast<const float4 *>(sb + at_col + i + k);
              v[k] = __fadd_rn(v[k], b4.x);
              v[k + 1] = __fadd_rn(v[k + 1], b4.y);
              v[k + 2] = __fadd_rn(v[k + 2], b4.z);
              v[k + 3] = __fadd_rn(v[k + 3], b4.w);
            }
          }
          if (!alive) {
#pragma unroll
            for (int k = 0; k < PER; ++k) v[k] = __int_as_float(0x7fffffff);
          }
          if constexpr (sizeof(T) == 4)
            word[i / PER] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
          else
            word[i / PER] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();  // the block is free again
        // row `lane` of the block: its eight 16-byte words lie where the 128-byte swizzle has them
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4 *>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = word[i];
        if (n_tile + c0 + CW <= p.tma_cols) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&tmC),
                         "r"(smem_u32(stage)), "r"(n_tile + c0), "r"(m0)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {  // rows of any alignment, and the end of a row: a row of the block at a time, its columns side by side
          __syncwarp();
          const int rows = min(32, p.M - m0), n_in = min(CW, p.N - n_tile - c0);
          for (int r = 0; r < rows; ++r) {
            T *out = (T *)p.o.p + (int64_t)(m0 + r) * p.o.ld + n_tile + c0;
#pragma unroll
            for (int j = 0; j < CW / 32; ++j) {
              const int c = j * 32 + lane;
              const T *from = reinterpret_cast<const T *>(stage + r * 128 + (((c / PER_WORD<T>) ^ (r & 7)) << 4)) + c % PER_WORD<T>;
              if (c < n_in) out[c] = *from;
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2 && rank != 0)
          asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(tempty_bar(a), 0))
                       : "memory");
        else
          mbar_arrive(tempty_bar(a));
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort) {
    if (threadIdx.x == 0 && rank == 0) drain_fills(full_bar, STAGES, issued, s, ph);
    if (threadIdx.x == 0 && rank != 0) {  // its copies count at the first CTA's barriers; they take some microseconds
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {}
    }
    if (threadIdx.x == 32 && issued) {
      commit<CG>(drain_bar);
      drain_products(drain_bar);
    }
    __syncthreads();
  }
  if (CG == 2) cluster_sync();  // nothing of the pair is at work in this CTA's memory any more
  tc_fence_after();
  if (warp == 1) {
    if (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
  }
}

// ------------------------------------------------------------------ few tokens
// One tile of up to 128 tokens x bn channels per cluster, its K split over the cluster's CTAs, so that as many SMs as there
// are stream w and most of a CTA's copies are in flight at once; each CTA's int32 sums go to its shared memory, and the
// cluster adds them there (exact in any order).  Bound by latency: 64 x 4096 -> 2048 6.5 us (8.4 MB of w: 1.3 us), 32 x 2048 ->
// 8192 7.1 (16.8 MB: 2.6).
constexpr int SPLIT_THREADS = 64 + 32 * EPI_WARPS;  // TMA, MMA and epilogue warps; all of them add
constexpr int SPLIT_RING = 108 * 1024;  // two CTAs fit an SM: the next call's are set up while this one's work
constexpr int SPLIT_MAX_STAGES = 24;
constexpr int SPLIT_SCALES = SPLIT_RING, SPLIT_BARS = SPLIT_SCALES + 3 * 128 * 4;
constexpr int SPLIT_SMEM = SPLIT_BARS + 512 + 1024;

struct SplitParams {
  Out o;
  int M, N, K;
  int bn, a_rows, stages, slot, split, tiles_n;
  int vec_out;
  uint32_t idesc;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ int4 ld_cluster(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__global__ void __launch_bounds__(SPLIT_THREADS, 1)
    int8_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const SplitParams p) {
  extern __shared__ __align__(1024) unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;  // the same in all CTAs of a cluster
  unsigned char *gbase = smem_dyn + (base - raw);
  const uint32_t bar0 = base + SPLIT_BARS;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (SPLIT_MAX_STAGES + s); };
  const uint32_t done_bar = bar0 + 8u * (2 * SPLIT_MAX_STAGES);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(gbase + SPLIT_BARS + 8 * (2 * SPLIT_MAX_STAGES + 1));
  volatile int *abort = reinterpret_cast<volatile int *>(gbase + SPLIT_BARS + 8 * (2 * SPLIT_MAX_STAGES + 1) + 8);
  const uint32_t abort_at = bar0 + 8u * (2 * SPLIT_MAX_STAGES + 1) + 8u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int tile = (int)(blockIdx.x / p.split), m0 = tile / p.tiles_n * BM, n0 = tile % p.tiles_n * p.bn;
  const int rows = min(BM, p.M - m0);
  const int num_kb = (p.K + BK - 1) / BK;
  const int kb0 = (int)((long)num_kb * rank / p.split), kb1 = (int)((long)num_kb * (rank + 1) / p.split);

  if (threadIdx.x == 0) {
    // w on its way to L2 (where a write of the kernel before would meet it) while that kernel ends
    for (int kb = kb0; kb < kb1 && kb < kb0 + p.stages; ++kb)
      asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&tmB), "r"(kb * BK), "r"(n0)
                   : "memory");
    for (int s = 0; s < p.stages && s < kb1 - kb0; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_u32(tmem_holder)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before the tensor memory is there: a next kernel's CTA that took it first, and waits for this kernel, would end both.
  MTP_PDL_TRIGGER();
  MTP_PDL_WAIT();
  const uint32_t tmem_base = *tmem_holder;
  constexpr int LD_PART = 132;  // of a token's sums, in words: 16-byte writes of a warp's rows meet each bank equally often
  int *part = reinterpret_cast<int *>(gbase);
  int s = 0, issued = 0;  // of the threads that issue copies and products: the ring's next slot, its parity, fills issued
  uint32_t ph = 0;
  float *scale_w = reinterpret_cast<float *>(gbase + SPLIT_SCALES), *bias_w = scale_w + 128, *scale_a = scale_w + 256;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t tx_bytes = (uint32_t)((p.a_rows + p.bn) * BK);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb >= kb0 + p.stages && !mbar_wait(empty_bar(s), ph ^ 1u, abort, p.timeout_ns)) break;
        mbar_expect_tx(full_bar(s), tx_bytes);
        const uint32_t sa = base + s * p.slot;
        tma_load_2d(sa, &tmA, full_bar(s), kb * BK, m0);
        tma_load_2d(sa + p.a_rows * BK, &tmB, full_bar(s), kb * BK, n0);
        ++issued;
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full_bar(s), ph, abort, p.timeout_ns)) break;
        tc_fence_after();
        const uint32_t sa = base + s * p.slot;
        const uint64_t ad = sw128_desc(sa), bd = sw128_desc(sa + p.a_rows * BK);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma<1>(tmem_base, ad + (uint64_t)(2 * k), bd + (uint64_t)(2 * k), p.idesc, (kb > kb0) || k != 0);
        commit<1>(empty_bar(s));
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      commit<1>(done_bar);  // after an expired wait for what has been issued
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    if (threadIdx.x - 64 < 128) {  // the scales come while the sums are made
      const int i = threadIdx.x - 64;
      const bool in = i < p.bn && n0 + i < p.N;
      scale_w[i] = in ? p.o.w_scale[n0 + i] : 0.f;
      bias_w[i] = in ? ld_bias(p.o, n0 + i) : 0.f;
      scale_a[i] = i < rows ? p.o.a_scale[m0 + i] : 0.f;
    }
    const bool alive = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort, p.timeout_ns + p.timeout_ns / 2));
    tc_fence_after();
    if (alive && q * 32 < rows) {
      const int m = q * 32 + lane;
      for (int c = 32 * half; c < p.bn; c += 64) {
        int r[32];
        tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (m < rows) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            if (c + i < p.bn)
              *reinterpret_cast<int4 *>(part + m * LD_PART + c + i) = make_int4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  {
    const int quads = p.bn / 4;
    bool lost = false;
    for (int i = 0; i < p.split; ++i) {
      int v;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(abort_at, i)));
      lost |= v != 0;
    }
    // a warp takes a row of sums, or two or four where they are short, of every split-th block of rows
    const int fold = quads <= 8 ? 2 : quads <= 16 ? 1 : 0, per = 1 << fold;
    const int c = (lane & (31 >> fold)) * 4, n = n0 + c;
    for (int m = (((int)rank * (SPLIT_THREADS / 32) + warp) << fold) + (lane >> (5 - fold)); m < rows;
         m += p.split * (SPLIT_THREADS / 32) * per) {
      if (c >= p.bn || n >= p.N) continue;
      const uint32_t at = base + (uint32_t)(m * LD_PART + c) * 4u;
      int4 part_of[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < p.split) part_of[i] = ld_cluster(cluster_addr(at, i));
      int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= p.split) continue;
        sum.x += part_of[i].x; sum.y += part_of[i].y; sum.z += part_of[i].z; sum.w += part_of[i].w;
      }
      const float sa = scale_a[m];
      const int in = min(4, p.N - n);
      float y[4] = {(float)sum.x, (float)sum.y, (float)sum.z, (float)sum.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = __fmul_rn(__fmul_rn(y[i], sa), scale_w[c + i]);
        if (p.o.bias) y[i] = __fadd_rn(y[i], bias_w[c + i]);
        if (lost) y[i] = __int_as_float(0x7fffffff);
      }
      if (p.vec_out && in == 4) {
        const int64_t to = (int64_t)(m0 + m) * p.o.ld + n;
        if (p.o.dtype == MTP_F32) *reinterpret_cast<float4 *>((float *)p.o.p + to) = make_float4(y[0], y[1], y[2], y[3]);
        else if (p.o.dtype == MTP_BF16)
          *reinterpret_cast<uint2 *>((__nv_bfloat16 *)p.o.p + to) = make_uint2(pack2<__nv_bfloat16>(y[0], y[1]), pack2<__nv_bfloat16>(y[2], y[3]));
        else *reinterpret_cast<uint2 *>((__half *)p.o.p + to) = make_uint2(pack2<__half>(y[0], y[1]), pack2<__half>(y[2], y[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < in) store_value(p.o, m0 + m, n + i, y[i]);
      }
    }
  }
  if (*abort) {
    if (threadIdx.x == 0) drain_fills(full_bar, p.stages, issued, s, ph);
    if (threadIdx.x == 32) drain_products(done_bar);
    __syncwarp();
  }
  // No other CTA reads this one's sums any more.  (Relaxed: nothing written since is read in the cluster; a release would wait
  // for the results' stores, 0.8 us.)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem_base));
}

// 2-D map over bytes [rows, cols] with ld bytes between rows; boxes of 128 bytes x box_rows, zeros outside.
int map_codes(CUtensorMap *tm, const void *ptr, int rows, int cols, int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MTP_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  if (rows == 1) ld = (cols + 15) / 16 * 16;  // not used
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(ptr), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MTP_ERR_ARG, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return MTP_OK;
}

// The same over the results; boxes of 128 bytes x 32 rows.
int map_out(CUtensorMap *tm, const Out &o, int rows, int cols) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MTP_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int es = o.dtype == MTP_F32 ? 4 : 2;
  const int64_t ld = rows == 1 ? ((int64_t)cols * es + 15) / 16 * 16 : o.ld * es;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32u};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = o.dtype == MTP_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : o.dtype == MTP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = fn(tm, type, 2, o.p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MTP_ERR_ARG, "cuTensorMapEncodeTiled (out) failed with code " + std::to_string((int)r));
  return MTP_OK;
}

// The kernel's limit of shared memory belongs to the current device.
template <int CG, typename T> int allow_smem() {
  static std::atomic<uint64_t> done{0};  // a bit for each device
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load() & bit) return MTP_OK;
  if (cudaFuncSetAttribute(int8_tc_kernel<CG, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) {
    cudaGetLastError();
    return fail(MTP_ERR_CUDA, "int8_tc: shared memory");
  }
  done.fetch_or(bit);
  return MTP_OK;
}

template <int CG, typename T>
int launch(const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &tcm, const Params &p, cudaStream_t stream) {
  int rc = allow_smem<CG, T>();
  if (rc) return rc;
  const int places = num_sms() / CG;
  const int grid = (p.num_tiles < places ? p.num_tiles : places) * CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, int8_tc_kernel<CG, T>, ta, tb, tcm, p);
  return check_launch("int8_linear");
}

template <int CG> Params tile_params(int M, int K, int N, const Out &o, int bn) {
  Params p{};
  p.o = o;
  p.M = M;
  p.N = N;
  p.K = K;
  p.bn = bn;
  p.tiles_m = ceil_div(M, BM * CG);
  p.tiles_n = ceil_div(N, bn);
  p.num_tiles = p.tiles_m * p.tiles_n;
  p.group_m = 16;
  auto inverse = [](int64_t n) { return n > 1 ? ~(uint64_t)0 / (uint64_t)n + 1 : 0; };
  p.div_group = inverse((int64_t)p.group_m * p.tiles_n);
  p.div_m = inverse(p.group_m);
  p.div_last = inverse(p.tiles_m % p.group_m);
  // kind::i8, int32 results, signed operands, both with K innermost
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(BM * CG >> 4) << 24);
  const size_t es = o.dtype == MTP_F32 ? 4 : 2;
  // a TMA store writes whole words of 16 bytes, past the end of a row that ends inside one
  if (aligned16(o.p) && (M == 1 || ((size_t)o.ld * es) % 16 == 0)) p.tma_cols = N * es % 16 == 0 ? 0x7fffffff : N;
  p.timeout_ns = TIMEOUT_NS;
  return p;
}

template <int CG>
int run(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o, int bn,
        cudaStream_t stream) {
  const Params p = tile_params<CG>(M, K, N, o, bn);
  CUtensorMap ta, tb, tcm;
  int rc = map_codes(&ta, a, M, K, ld_a, BM);
  if (rc) return rc;
  rc = map_codes(&tb, w, N, K, ld_w, bn / CG);
  if (rc) return rc;
  memset(&tcm, 0, sizeof(tcm));
  if (p.tma_cols) {
    rc = map_out(&tcm, o, M, N);
    if (rc) return rc;
  }
  if (o.dtype == MTP_F32) return launch<CG, float>(ta, tb, tcm, p, stream);
  if (o.dtype == MTP_BF16) return launch<CG, __nv_bfloat16>(ta, tb, tcm, p, stream);
  return launch<CG, __half>(ta, tb, tcm, p, stream);
}

// The kernel's limit of shared memory belongs to the current device.
int allow_split_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load() & bit) return MTP_OK;
  if (cudaFuncSetAttribute(int8_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SPLIT_SMEM) != cudaSuccess) {
    cudaGetLastError();
    return fail(MTP_ERR_CUDA, "int8_split: shared memory");
  }
  done.fetch_or(bit);
  return MTP_OK;
}

// The split with the least time, and that time in us by what was measured: a call takes 4.4, a CTA's bytes come at 62 KB/us
// (64 x 2048 -> 8192 in one, 256 KB: 8.7; 64 x 4096 -> 2048 in four, 131 KB: 6.5, in one, 524 KB: 12.2), the addition takes
// 0.5, a further wave 2.
double plan_split(int M, int N, int K, int &split_of_k, int &columns) {
  const int sms = num_sms(), num_kb = ceil_div(K, BK), tiles_m = ceil_div(M, BM);
  const int a_rows = M < BM ? (M + 7) / 8 * 8 : BM;
  double best = 1e30;
  for (int split = 1; split <= 8 && split <= num_kb; split *= 2) {
    int bn = (ceil_div((int64_t)N * split * tiles_m, sms) + 15) / 16 * 16;
    bn = bn < 32 ? 32 : bn > 128 ? 128 : bn;
    const int64_t waves = ((int64_t)ceil_div(N, bn) * tiles_m * split + sms - 1) / sms;
    const double kb = (double)ceil_div(num_kb, split) * (bn + a_rows) * BK / 1e3;
    const double time = 4.4 + (double)waves * kb / 62.0 + (double)(waves - 1) * 2.0 + (split > 1 ? 0.5 : 0.0);
    if (time < best) {
      best = time;
      split_of_k = split;
      columns = bn;
    }
  }
  return best;
}

SplitParams split_params(int M, int K, int N, const Out &o, int split, int bn) {
  SplitParams p{};
  p.o = o;
  p.M = M;
  p.N = N;
  p.K = K;
  p.a_rows = M < BM ? (M + 7) / 8 * 8 : BM;
  p.split = split;
  p.bn = bn;
  p.tiles_n = ceil_div(N, bn);
  p.slot = (p.a_rows + p.bn) * BK;
  // rows of tokens past a_rows are read by the tensor core from what follows in the slot: the last slot ends 128 rows in
  p.stages = (SPLIT_RING - (BM - p.a_rows) * BK) / p.slot;
  if (p.stages > SPLIT_MAX_STAGES) p.stages = SPLIT_MAX_STAGES;
  p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  const size_t es = o.dtype == MTP_F32 ? 4 : 2;
  p.vec_out = aligned(o.p, 4 * es) && (M == 1 || o.ld % 4 == 0);
  p.timeout_ns = TIMEOUT_NS;
  return p;
}

int launch_split(const CUtensorMap &ta, const CUtensorMap &tb, const SplitParams &p, cudaStream_t stream) {
  int rc = allow_split_smem();
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ceil_div(p.M, BM) * p.tiles_n * p.split);
  cfg.blockDim = dim3(SPLIT_THREADS);
  cfg.dynamicSmemBytes = SPLIT_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, int8_split_kernel, ta, tb, p);
  return check_launch("int8_linear");
}

int run_split(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o, int split, int bn,
              cudaStream_t stream) {
  const SplitParams p = split_params(M, K, N, o, split, bn);
  CUtensorMap ta, tb;
  int rc = map_codes(&ta, a, M, K, ld_a, p.a_rows);
  if (rc) return rc;
  rc = map_codes(&tb, w, N, K, ld_w, p.bn);
  if (rc) return rc;
  return launch_split(ta, tb, p, stream);
}

}  // namespace

bool tc_eligible(const int8_t *a, int64_t ld_a, int M, const int8_t *w, int64_t ld_w, int N) {
  return aligned16(a) && aligned16(w) && (M == 1 || ld_a % 16 == 0) && (N == 1 || ld_w % 16 == 0) && M < 0x7ffff000 &&
         N < 0x7ffff000;
}

int linear_tc(const int8_t *a, int64_t ld_a, int M, int K, const int8_t *w, int64_t ld_w, int N, const Out &o,
              cudaStream_t stream) {
  // Of three tiles the one with the least time by what was measured (us): a call's own, then for each round of tiles 0.3 for a
  // block of K, whatever the tile, and what the epilogue adds.  (512 x 2048 -> 8192: 22.4, 14.1 and 11.7 us; 256 rows: 13.2,
  // 9.2 and 11.3; 256 x 2048 -> 1024: 7.7, 8.2 and 9.9.)
  const int sms = num_sms(), num_kb = ceil_div(K, BK);
  auto time_of = [&](int cg, int bn, double call, double kb, double tile) {
    const int64_t tiles = (int64_t)ceil_div(M, BM * cg) * ceil_div(N, bn), places = sms / cg;
    return call + (double)((tiles + places - 1) / places) * (num_kb * kb + tile);
  };
  const double t1 = time_of(1, 64, 2.3, 0.287, 0.42), t2 = time_of(1, 128, 2.3, 0.287, 1.1), t3 = time_of(2, 256, 3.4, 0.306, 1.6);
  if (M <= 2 * BM) {
    // Below 64 rows by split K (32 x 2048 -> 8192: 7.1 us, by tiles of 64 columns 10.6); from there where it is the faster (128
    // x 2048 -> 8192: 9.4 and 8.5; 128 x 4096 -> 2048: 7.7 and 12.1; 160 x 4096 -> 2048: 10.8 and 12.3).
    int split = 1, bn = 128;
    const double t = plan_split(M, N, K, split, bn);
    if (M < 64 || t <= (t1 < t2 ? t1 : t2) + 0.5) return run_split(a, ld_a, M, K, w, ld_w, N, o, split, bn, stream);
  }
  if (M > BM && t3 <= t1 && t3 <= t2) return run<2>(a, ld_a, M, K, w, ld_w, N, o, 256, stream);
  return run<1>(a, ld_a, M, K, w, ld_w, N, o, t2 <= t1 ? 128 : 64, stream);
}

}  // namespace i8
}  // namespace mtp

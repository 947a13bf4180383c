// Operators on logits rows: the log probability of a given token with entropy and top alternatives, its gradient, and
// the distillation loss from a teacher's top logits with its gradient.
//
// With z = x / T, m = max z and S = sum e^(z - m), a row gives
//   log p_j = (z_j - m) - log S          H = log S - sum e^(z - m) (z - m) / S
// All sums and statistics are fp32.  A row belongs to a group of threads: a warp (short rows, eight to a CTA), a CTA, or
// a cluster of up to 8 CTAs (few rows).  A row is read in 16-byte vectors at its own alignment (the elements before the
// first and after the last whole vector one by one), through a ring in shared memory that asynchronous copies fill: a
// thread reads only what it copied itself, so that nothing waits for another thread.  A forward pass reads its row once:
// each thread keeps the running maximum m, S and U = sum e^y y (y in units of log2) of its elements and rescales them
// when m grows; threads and CTAs are joined at the end.  A pass that needs the row a second time takes it in the opposite
// order: first what is still in the ring, then the part of the row that L2 saw last.
#include <cooperative_groups.h>
#include "common.cuh"
#include "logits.cuh"

namespace mtp {
namespace {

namespace cg = cooperative_groups;
using namespace lg;

constexpr int MAX_TOP = 128;      // alternatives or teacher entries per row
constexpr int CTA = 256;          // threads per CTA
constexpr int MAX_CLUSTER = 8;    // CTAs that share a row
constexpr int RING = 4;           // pairs of vectors per thread in flight: 32 KB a CTA
constexpr int RING_BYTES = 2 * RING * CTA * 16;

// The threads that share a row within a CTA: GW warps.
template <int GW> struct Group {
  static_assert(GW == 1 || GW == CTA / 32, "a warp or the CTA");
  static constexpr int NT = 32 * GW, ROWS = CTA / NT;  // threads of the group, groups of the CTA
  static __device__ __forceinline__ int tid() { return threadIdx.x & (NT - 1); }
  static __device__ __forceinline__ int index() { return threadIdx.x / NT; }
  static __device__ __forceinline__ void sync() {
    if (GW == 1) __syncwarp();
    else __syncthreads();
  }
};

// Row r of a batch laid out as [outer][inner] rows: r = o * inner + i; inner 0: one level, r = i.  (Integer divisions are
// what a thread's fixed cost per row consists of, so they are few and of 32 bits.)
struct Rows {
  uint32_t inner;
  int64_t ld_outer, ld;
  __device__ __forceinline__ int64_t at(uint32_t r) const {
    if (inner == 0) return r * ld;
    const uint32_t o = r / inner;
    return o * ld_outer + (r - o * inner) * ld;
  }
};
inline Rows make_rows(int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld) {
  if (outer == 1) return Rows{0, 0, ld};
  if (inner == 1) return Rows{0, 0, ld_outer};
  return Rows{(uint32_t)inner, ld_outer, ld};
}

// The calling thread's row, and which of the 2^shift CTAs that share it this one is.
template <int GW> struct Part {
  uint32_t row;
  int rank, shift;
  __device__ __forceinline__ explicit Part(int s)
      : row(GW == 1 ? blockIdx.x * Group<1>::ROWS + Group<1>::index() : blockIdx.x >> s),
        rank(GW == 1 ? 0 : (int)(blockIdx.x & ((1u << s) - 1))), shift(GW == 1 ? 0 : s) {}
};

// ----------------------------------------------------------------- rows in vectors
// 16 bytes of logits.
template <typename T> struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4 &r, float (&x)[N]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(x[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ uint4 load16(const void *p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// The part of a row that CTA `rank` of 2^shift works on: vectors [v0, v1) of those that start `head` elements into the
// row, the first CTA also the elements before them, the last the `tail` elements from `tail0` on.  Thread t of the group
// takes the vectors v0 + t, v0 + t + NT, ... (n of them), and one of the elements at each end.
template <typename T, int GW> struct Slice {
  static constexpr int N = Vec<T>::N, NT = Group<GW>::NT, STEP = NT * N;  // STEP: elements between a thread's vectors
  const T *row;
  int head, v0, v1, nhead, tail0, ntail, n;
  __device__ __forceinline__ Slice(const T *r, int V, int rank, int shift) : row(r) {
    head = (int)(((16u - (unsigned)(reinterpret_cast<uintptr_t>(r) & 15u)) & 15u) / sizeof(T));
    if (head > V) head = V;
    const int nv = (V - head) / N;
    v0 = (int)((int64_t)nv * rank >> shift);
    v1 = (int)((int64_t)nv * (rank + 1) >> shift);
    nhead = rank == 0 ? head : 0;
    tail0 = head + nv * N;
    ntail = rank + 1 == 1 << shift ? V - tail0 : 0;
    const int left = v1 - v0 - Group<GW>::tid();
    n = left > 0 ? (left + NT - 1) / NT : 0;
  }
  __device__ __forceinline__ const T *vec(int v) const { return row + head + (int64_t)v * N; }
  __device__ __forceinline__ int first(int v) const { return head + v * N; }  // index of a vector's first element
  __device__ __forceinline__ const T *mine() const { return vec(v0 + Group<GW>::tid()); }
  __device__ __forceinline__ int most() const { return (v1 - v0 + NT - 1) / NT; }  // n of the group's first thread
};

// Asynchronous 16-byte copies into the calling thread's own places of shared memory.
__device__ __forceinline__ void copy16(uint4 *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// A thread's places: pair p of its vectors is at [(p % RING) * 2 * NT] and NT further.  A group's part is contiguous.
template <int GW> __device__ __forceinline__ uint4 *ring_of(uint4 *ring) {
  constexpr int NT = Group<GW>::NT;
  return ring + Group<GW>::index() * 2 * RING * NT + Group<GW>::tid();
}
template <typename T, int GW>
__device__ __forceinline__ void fetch_pair(const Slice<T, GW> &sl, uint4 *mine, int p) {
  constexpr int NT = Group<GW>::NT;
  if (p >= 0 && 2 * p < sl.n) {
    uint4 *at = mine + (p % RING) * 2 * NT;
    const T *src = sl.mine() + (int64_t)(2 * p) * sl.STEP;
    copy16(at, src);
    if (2 * p + 1 < sl.n) copy16(at + NT, src + sl.STEP);
  }
  copy_commit();
}

// ----------------------------------------------------------------- row statistics
template <typename T, bool ENT, bool MASKED>
__device__ __forceinline__ float2 accumulate_pair(Stat &st, const uint4 &a, const uint4 &b, float c2, bool &masked) {
  constexpr int N = Vec<T>::N;
  float x[2 * N], lo[N], hi[N];
  Vec<T>::unpack(a, lo);
  Vec<T>::unpack(b, hi);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = lo[i], x[N + i] = hi[i];
  return accumulate<ENT, 2 * N, MASKED>(st, x, c2, masked);
}
template <typename T, bool ENT>
__device__ __forceinline__ float2 accumulate_vec(Stat &st, const uint4 &a, float c2) {
  float x[Vec<T>::N];
  Vec<T>::unpack(a, x);
  bool masked;
  const float2 mx = accumulate<ENT, Vec<T>::N, true>(st, x, c2, masked);
  return make_float2(fmaxf(mx.x, mx.y), -INFINITY);
}

// Maxima of a thread's chunks of `per` vectors (1, or a multiple of 2), for the alternatives: bf16, rounded up, at
// [chunk][thread].
constexpr int CHUNKS = 16;
struct ChunkMaxima {
  __nv_bfloat16 *at;
  int per;
};
template <typename T> __device__ __forceinline__ __nv_bfloat16 upper(float x) {
  return std::is_same<T, __nv_bfloat16>::value ? __float2bfloat16_rn(x) : __float2bfloat16_ru(x);
}

// One thread's statistics of its elements.  Afterwards the ring holds the thread's last RING pairs.
template <typename T, int GW, bool ENT, bool TOP>
__device__ __forceinline__ Stat thread_stats(const Slice<T, GW> &sl, float c2, uint4 *ring, ChunkMaxima cm) {
  constexpr int NT = Group<GW>::NT;
  Stat st{LOWEST, 0.f, 0.f};
  uint4 *mine = ring_of<GW>(ring);
#pragma unroll
  for (int p = 0; p < RING; ++p) fetch_pair(sl, mine, p);
  const int n = sl.n;
  const T *src = sl.mine() + (int64_t)2 * RING * sl.STEP;
  int slot = 0, in_chunk = 0, i = 0;
  bool masked = false;
  float chunk = -INFINITY;
  // Masked logits are many or none, as a rule, so a warp looks at its first pairs and then goes through one of two loops;
  // a thread that meets its first masked logit later changes over by itself.  777 rows of 50277 fp16 logits, a tenth of them
  // masked, seven alternatives 25.6 us; 29.5 with every thread changing over by itself, 29.0 with both forms in one loop, 34
  // with every group that holds a masked logit summed twice.  32 x 1023 unmasked rows of 50280 bf16 logits 662 us; 658, 668
  // and 654 (in another run).
  auto pairs = [&](auto after, int end) {
    constexpr bool MASKED = decltype(after)::value;
    while (i < end) {
      copy_wait<RING - 1>();
      uint4 *at = mine + slot * 2 * NT;
      const float2 mx = i + 1 < n ? accumulate_pair<T, ENT, MASKED>(st, at[0], at[NT], c2, masked)
                                  : accumulate_vec<T, ENT>(st, at[0], c2);
      if constexpr (TOP) {
        if (cm.per == 1) {
          cm.at[0] = upper<T>(mx.x);
          if (i + 1 < n) cm.at[CTA] = upper<T>(mx.y);
          cm.at += 2 * CTA;
        } else {
          chunk = max3(chunk, mx.x, mx.y);
          in_chunk += 2;
          if (in_chunk == cm.per) {
            *cm.at = upper<T>(chunk);
            cm.at += CTA;
            chunk = -INFINITY;
            in_chunk = 0;
          }
        }
      }
      if (i + 2 * RING < n) copy16(at, src);
      if (i + 2 * RING + 1 < n) copy16(at + NT, src + sl.STEP);
      copy_commit();
      src += 2 * sl.STEP;
      slot = (slot + 1) & (RING - 1);
      i += 2;
      if (ENT && !MASKED && masked) break;
    }
  };
  if constexpr (ENT) {
    pairs(std::false_type{}, min(n, 2));
    masked = __any_sync(0xffffffffu, masked);
    if (!masked) pairs(std::false_type{}, n);
    pairs(std::true_type{}, n);
  } else {
    pairs(std::false_type{}, n);
  }
  if constexpr (TOP) {
    if (in_chunk) *cm.at = upper<T>(chunk);
  }
  const int t = Group<GW>::tid();
  if (t < sl.nhead) accumulate1<ENT>(st, ldf(sl.row + t), c2);
  if (t < sl.ntail) accumulate1<ENT>(st, ldf(sl.row + sl.tail0 + t), c2);
  return st;
}

// Shared state of the CTAs of a row.  Every CTA gets every CTA's statistics (and group maxima) in its own copy.
struct RowShared {
  float m[CTA / 32];
  float2 su[CTA / 32];
  Stat cta[MAX_CLUSTER];
};

// A CTA of a cluster says that it runs and its shared memory may be written; the peers wait for that before they do.
__device__ __forceinline__ void cluster_begin(int parts) {
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_ready(int parts) {
  if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Joins the threads of the group and the CTAs of the cluster; every thread returns the row's statistics.  The maximum
// comes first, so that each thread rescales its sums once and the rest are additions, in an order that is the same in
// every thread.  Orders the shared memory written before it (the group maxima, peers' copies included) for all threads.
template <int GW, bool ENT>
__device__ __forceinline__ Stat row_join(Stat st, RowShared &sh, float c2, int rank, int parts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = warp_max(st.m);
  if constexpr (GW > 1) {
    if (lane == 0) sh.m[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GW; ++i) m = fmaxf(m, sh.m[i]);
  }
  const float y = fmaxf((st.m - m) * c2, FLOOR_Y), e = ex2(y);
  float u = ENT ? fmaf(y, st.s, st.u) * e : 0.f, s = st.s * e;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    if (ENT) u += __shfl_xor_sync(0xffffffffu, u, o);
  }
  Stat all{m, s, u};
  if constexpr (GW > 1) {
    if (lane == 0) sh.su[warp] = make_float2(s, u);
    __syncthreads();
    all.s = all.u = 0.f;
#pragma unroll
    for (int i = 0; i < GW; ++i) {
      all.s += sh.su[i].x;
      all.u += sh.su[i].y;
    }
    if (parts > 1) {
      cg::cluster_group cl = cg::this_cluster();
      if (threadIdx.x < (unsigned)parts) *cl.map_shared_rank(&sh.cta[rank], threadIdx.x) = all;
      cl.sync();
      all = sh.cta[0];
      for (int i = 1; i < parts; ++i) all = join<ENT>(all, sh.cta[i], c2);
    }
  }
  return all;
}

// ----------------------------------------------------------------- top alternatives
// Order of the alternatives as unsigned integers: larger value first, -0 equal to +0, NaN above +inf.  An element's
// key is its value's order above its complemented index, so that no two are equal and the lower index wins a tie.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = v == 0.f ? 0u : __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k == 0xFFFFFFFFu ? 0x7fffffffu : (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ uint64_t element_key(float v, int i) { return ((uint64_t)order_key(v) << 32) | (uint32_t)~i; }


// The k largest of a row without a second pass over it.  A lower bound of the k-th largest element is the k-th largest of
// the maxima of disjoint sets of elements: the threads of all CTAs in 256 sets (a set is `parts` neighbouring threads of
// a CTA), or for a warp's row the lanes' chunks.  Only chunks whose maximum reaches the bound are read again (k = 64 of
// 50280: about 75 of 4000); their elements that reach it go on the group's list.  The lists of a cluster are joined in its
// first CTA, and an element's place in the result is the number of elements above it.
template <int GW> struct TopShared {
  static constexpr int LIST = GW == 1 ? 384 : 1024;  // candidates
  static constexpr int JOINED = GW == 1 ? 0 : MAX_CLUSTER * MAX_TOP;  // the cluster's candidates
  static constexpr int WORK = GW == 1 ? 256 : 1024;  // chunks to be read again
  static_assert(8 * (LIST + JOINED) + 4 * WORK <= 2 * RING * Group<GW>::NT * 16, "they lie in the group's part of the ring");
  uint32_t set[GW == 1 ? 1 : CTA];  // order keys of the maxima of the sets, all CTAs'
  uint64_t red[GW];
  uint32_t bound;
  int n, work;
};

// Largest b with at least k of the warp's 32 * NK keys >= b, or a smaller one that at most k + k / 8 + 4 reach; the
// lowest key where all of them are fewer than k.
template <int NK> __device__ __forceinline__ uint32_t key_quantile(const uint32_t (&key)[NK], int k) {
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    lo = min(lo, key[i]);
    hi = max(hi, key[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  const int enough = k + k / 8 + 4;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    int c = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) c += key[i] >= mid;
    c = (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
    if (c >= k) {
      lo = mid;
      if (c <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// Calls f(value, index) for the calling thread's elements.
template <typename T, int GW, typename F>
__device__ __forceinline__ void thread_elements(const Slice<T, GW> &sl, F f) {
  constexpr int N = Vec<T>::N;
  const int t = Group<GW>::tid();
  for (int v = sl.v0 + t; v < sl.v1; v += Group<GW>::NT) {
    float x[N];
    Vec<T>::unpack(load16(sl.vec(v)), x);
#pragma unroll
    for (int i = 0; i < N; ++i) f(x[i], sl.first(v) + i);
  }
  if (t < sl.nhead) f(ldf(sl.row + t), t);
  if (t < sl.ntail) f(ldf(sl.row + sl.tail0 + t), sl.tail0 + t);
}

// Largest key that at least k of the group's counted elements reach, or a smaller one that at most `most` >= k reach.
// count(key): how many elements of the calling thread are >= key; lo: a key that at least k reach; no key is above hi.
template <int GW, typename F>
__device__ uint64_t key_bound(uint64_t lo, uint64_t hi, int k, int most, uint64_t *red, F count) {
  while (lo < hi) {
    const uint64_t mid = lo + (hi - lo) / 2 + 1;
    int c = (int)__reduce_add_sync(0xffffffffu, (unsigned)count(mid));
    if constexpr (GW > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = (uint64_t)c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < GW; ++i) c += (int)red[i];
    }
    if (c >= k) {
      lo = mid;
      if (c <= most) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// Cuts list[0, n) down to at most `most` >= k keys, the k largest among them; n <= LIST.
template <int GW> __device__ int cut_list(uint64_t *list, int n, int k, int most, TopShared<GW> &sh) {
  using G = Group<GW>;
  constexpr int EACH = (TopShared<GW>::LIST + G::NT - 1) / G::NT;
  if (n <= most) return n;
  const uint64_t b = key_bound<GW>(0, ~0ull, k, most, sh.red, [&](uint64_t key) {
    int c = 0;
    for (int i = G::tid(); i < n; i += G::NT) c += list[i] >= key;
    return c;
  });
  uint64_t mine[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = G::tid() + i * G::NT;
    mine[i] = at < n ? list[at] : 0;
  }
  G::sync();
  if (G::tid() == 0) sh.n = 0;
  G::sync();
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (mine[i] >= b && G::tid() + i * G::NT < n) list[atomicAdd(&sh.n, 1)] = mine[i];
  G::sync();
  return sh.n;
}

// st: the calling thread's own statistics, row: the row's; the maxima of the sets are in place (row_join has ordered
// them), and the ring has been read.
template <typename T, int GW>
__device__ __forceinline__ void top_alternatives(const Slice<T, GW> &sl, Stat st, RowStats row, int k, float inv_t, int V,
                                                 TopShared<GW> &sh, uint4 *ring, ChunkMaxima cm, int rank, int parts,
                                                 int64_t *ids, float *logprobs) {
  using G = Group<GW>;
  using S = TopShared<GW>;
  constexpr int NT = G::NT, N = Vec<T>::N;
  const int t = G::tid(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t *list = reinterpret_cast<uint64_t *>(ring + G::index() * 2 * RING * NT);
  int *work = reinterpret_cast<int *>(list + S::LIST + S::JOINED);
  const int chunks = (sl.n + cm.per - 1) / cm.per;  // the calling thread's
  uint32_t bound;
  if constexpr (GW == 1) {
    // a maximum that was rounded up is at least the next lower bf16
    constexpr uint32_t down = std::is_same<T, __nv_bfloat16>::value ? 0u : 0x10000u;
    uint32_t key[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) key[c] = c < chunks ? order_key(__bfloat162float(cm.at[c * CTA])) - down : 0u;
    bound = key_quantile<CHUNKS>(key, k);
    if (lane == 0) sh.n = sh.work = 0;
  } else {
    if (warp == 0) {
      uint32_t key[CTA / 32];
#pragma unroll
      for (int i = 0; i < CTA / 32; ++i) key[i] = sh.set[lane + 32 * i];
      const uint32_t b = key_quantile<CTA / 32>(key, k);
      if (lane == 0) {
        sh.bound = b;
        sh.n = sh.work = 0;
      }
    }
    __syncthreads();
    bound = sh.bound;
  }
  const float least = key_value(bound);  // below every order (a set without an element) it is NaN, which all pass
  auto take = [&](float x, int i) {
    if (!(x < least)) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < S::LIST) list[at] = element_key(x, i);
    }
  };
  G::sync();
  // a thread whose sum is NaN may hold a NaN, which maxima pass over
  const bool nan = st.s != st.s;
  if (nan || !(st.m < least) || st.s == 0.f) {
    for (int c = 0; c < chunks; ++c) {
      if (nan || !(__bfloat162float(cm.at[c * CTA]) < least)) {
        const int at = atomicAdd(&sh.work, 1);
        if (at < S::WORK) work[at] = t * CHUNKS + c;
      }
    }
    if (t < sl.nhead) take(ldf(sl.row + t), t);
    if (t < sl.ntail) take(ldf(sl.row + sl.tail0 + t), sl.tail0 + t);
  }
  G::sync();
  const int items = sh.work;
  if (items <= S::WORK) {
    for (int e = t; e < items; e += NT) {
      const int of = work[e] / CHUNKS, first = sl.v0 + of + cm.per * (work[e] % CHUNKS) * NT;
      for (int j = 0; j < cm.per; j += 2) {
        const int v = first + j * NT;
        if (v >= sl.v1) break;
        const bool two = cm.per > 1 && v + NT < sl.v1;
        const uint4 a = load16(sl.vec(v)), b = two ? load16(sl.vec(v + NT)) : make_uint4(0, 0, 0, 0);
        float x[N];
        Vec<T>::unpack(a, x);
#pragma unroll
        for (int i = 0; i < N; ++i) take(x[i], sl.first(v) + i);
        if (two) {
          Vec<T>::unpack(b, x);
#pragma unroll
          for (int i = 0; i < N; ++i) take(x[i], sl.first(v + NT) + i);
        }
      }
    }
  }
  G::sync();
  int n = sh.n;
  if (n > S::LIST || items > S::WORK) {
    // more elements reach the bound than the list holds (a row of equal logits): find the key of this CTA's k-th
    // largest element by bisection, one scan of the slice a step, and collect again
    const uint64_t lo = ((uint64_t)bound << 32) | (uint32_t)~(V - 1);
    const uint64_t hi = row.log_s != row.log_s ? ~0ull : ((uint64_t)order_key(row.m) << 32) | 0xFFFFFFFFu;
    const uint64_t b = key_bound<GW>(lo, hi, k, MAX_TOP, sh.red, [&](uint64_t key) {
      int c = 0;
      thread_elements(sl, [&](float x, int i) { c += element_key(x, i) >= key; });
      return c;
    });
    G::sync();
    if (t == 0) sh.n = 0;
    G::sync();
    thread_elements(sl, [&](float x, int i) {
      const uint64_t key = element_key(x, i);
      if (key >= b) list[atomicAdd(&sh.n, 1)] = key;
    });
    G::sync();
    n = sh.n;
  }
  if constexpr (GW > 1) {
    if (parts > 1) {
      n = cut_list<GW>(list, n, k, MAX_TOP, sh);
      __syncthreads();
      if (t == 0) sh.n = n;
      cg::cluster_group cl = cg::this_cluster();
      cl.sync();
      if (rank == 0) {
        int at = 0;
        for (int c = 0; c < parts; ++c) {
          const int nc = *cl.map_shared_rank(&sh.n, c);
          const uint64_t *from = cl.map_shared_rank(list, c);
          if (t < nc) list[S::LIST + at + t] = from[t];
          at += nc;
        }
        n = at;
      }
      cl.sync();  // the peers' lists have been read
      if (rank != 0) return;
      list += S::LIST;
    }
    n = cut_list<GW>(list, n, k, 2 * MAX_TOP, sh);
  }
  for (int e = t; e < n; e += NT) {
    const uint64_t key = list[e];
    int place = 0;
    for (int i = 0; i < n; ++i) place += list[i] > key;
    if (place < k) {
      ids[place] = (int64_t)(int)~(uint32_t)key;
      logprobs[place] = log_prob(key_value((uint32_t)(key >> 32)), row.m, row.log_s, inv_t);
    }
  }
}

// ----------------------------------------------------------------- log probabilities
// Bound by the exponentials at the clocks of a long run under the power cap (16 per cycle and SM, 1.06 a logit: 480 us of
// the 655 us that 32 x 1023 rows of 50280 bf16 logits take at 1.53 GHz, their issue slots 75% used), by HBM otherwise: the
// same rows 568 us in isolation, 5.80 TB/s or 0.90 of the measured copy rate.  fp32 rows are HBM-bound: 4096 of 50280
// 139 us, 0.92.  A ring of 32 KB per CTA and five CTAs per SM were taken: 6 CTAs (spills) 575 us, a ring twice as deep
// (three CTAs) 11% slower.  Alternatives cost a row its joins and the second look: 2048 fp32 rows 98 us with 64 of them.
struct FwdArgs {
  const int64_t *targets;
  float *logprob, *entropy, *stats;
  int top_k;
  int64_t *top_ids;
  float *top_logprobs;
  float inv_t, c2;  // 1 / T, log2 e / T
  int V, shift;
  uint32_t rows;
  const int *expired;  // of fp32 logits: a word that is set if a wait of the pass that made them has expired, or null
};

template <typename T, int GW, bool ENT, bool TOP>
__global__ void __launch_bounds__(CTA, GW == 1 ? 4 : 5) token_logprobs_kernel(const T *__restrict__ logits, Rows rows, FwdArgs a) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  using G = Group<GW>;
  extern __shared__ uint4 ring[];
  __shared__ RowShared sh;
  __shared__ TopShared<GW> top[G::ROWS];
  __shared__ __nv_bfloat16 maxima[TOP ? CHUNKS * CTA : 1];
  const Part<GW> part(a.shift);
  if (GW == 1 && part.row >= a.rows) return;
  const int parts = 1 << part.shift, rank = part.rank;
  const int64_t r = part.row;
  const T *row = logits + rows.at(part.row);
  const Slice<T, GW> sl(row, a.V, rank, part.shift);
  const ChunkMaxima cm{maxima + (TOP ? threadIdx.x : 0),
                       !TOP || sl.most() <= CHUNKS ? 1 : (sl.most() + 2 * CHUNKS - 1) / (2 * CHUNKS) * 2};
  cluster_begin(parts);
  const Stat st = thread_stats<T, GW, ENT, TOP>(sl, a.c2, ring, cm);
  cluster_ready(parts);
  if constexpr (TOP && GW > 1) {
    // maxima of the sets of `parts` threads to every CTA of the cluster
    uint32_t g = sl.n > 0 || G::tid() < sl.nhead || G::tid() < sl.ntail ? order_key(st.s == 0.f ? -INFINITY : st.m) : 0u;
    for (int o = 1; o < parts; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    const int slot = rank * (CTA >> part.shift) + ((int)threadIdx.x >> part.shift);
    if (parts > 1) *cg::this_cluster().map_shared_rank(&top[0].set[slot], threadIdx.x & (parts - 1)) = g;
    else top[0].set[slot] = g;
  }
  const Stat all = row_join<GW, ENT>(st, sh, a.c2, rank, parts);
  if (!TOP && threadIdx.x >= 32 && GW > 1) return;
  RowStats s = finish(all);
  if (std::is_same<T, float>::value && a.expired && *a.expired) s = expired();
  if (rank == 0 && G::tid() == 0) {
    if (a.logprob) {
      const int64_t t = a.targets[r];
      a.logprob[r] = t < 0 ? 0.f : t >= a.V ? NAN : log_prob(ldf(row + t), s.m, s.log_s, a.inv_t);
    }
    if (a.entropy) a.entropy[r] = s.entropy;
    if (a.stats) {
      a.stats[2 * r] = s.m;
      a.stats[2 * r + 1] = s.log_s;
    }
  }
  if constexpr (TOP)
    top_alternatives<T, GW>(sl, st, s, a.top_k, a.inv_t, a.V, top[G::index()], ring, cm, rank, parts,
                            a.top_ids + r * a.top_k, a.top_logprobs + r * a.top_k);
}

// ----------------------------------------------------------------- gradients
// out_j = p_j (a + b y_j) with p_j = 2^y_j, y = log2 p; the element `hit` gets `extra` on top.  ENT: b is not 0.
// A p below 2^-126 still counts where its factor is large: 2^(y + 32) is taken, which is flushed to zero only where p
// is below the smallest subnormal, and 2^-32 goes into the factor.  Where the factor is below 2^-29 its product with such
// a p vanishes anyway, and 2^-32 might push the factor itself out of range: there the lift is 0.
template <bool ENT> struct Dense {
  float m, l2, c2;  // largest logit, log2 S (less the lift, if not ENT), log2 e / T
  float a, b, lift;  // a and b times 2^-lift
  __device__ __forceinline__ Dense(float m_, float log_s, float c2_, float a_, float b_)
      : m(m_), l2(log_s * LOG2E), c2(c2_), a(a_), b(b_), lift(0.f) {
    if (!(fmaxf(fabsf(a), ENT ? -FLOOR_Y * fabsf(b) : 0.f) < 0x1p-30f)) {
      lift = 32.f;
      a *= 0x1p-32f;
      b *= 0x1p-32f;
    }
    if (!ENT) l2 -= lift;
  }
  __device__ __forceinline__ F2 two(F2 x) const {
    const F2 y = fma2(add2(x, f2(-m, -m)), f2(c2, c2), f2(-l2, -l2));
    float y0, y1;
    if constexpr (!ENT) {
      un2(y, y0, y1);
      return mul2(f2(ex2(y0), ex2(y1)), f2(a, a));
    } else {
      un2(y, y0, y1);
      const F2 f = fma2(f2(fmaxf(y0, FLOOR_Y), fmaxf(y1, FLOOR_Y)), f2(b, b), f2(a, a));
      un2(add2(y, f2(lift, lift)), y0, y1);
      return mul2(f2(ex2(y0), ex2(y1)), f);
    }
  }
  __device__ __forceinline__ float one(float x) const {
    float v, w;
    un2(two(f2(x, x)), v, w);
    return v;
  }
};

// Writes the slice's gradient, last pair first.  KEPT: thread_stats has just read the slice, so the ring holds the
// thread's last RING pairs.  16-byte stores where the gradient row is aligned as the logits row is.
template <typename T, int GW, bool KEPT, bool ENT>
__device__ __forceinline__ void write_grad(const Slice<T, GW> &sl, T *out, const Dense<ENT> &d, bool zero, int64_t hit,
                                           float extra, uint4 *ring) {
  constexpr int N = Vec<T>::N, NT = Group<GW>::NT;
  const bool same = ((reinterpret_cast<uintptr_t>(sl.row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  const int t = Group<GW>::tid();
  auto one = [&](int i) {
    float v = 0.f;
    if (!zero) {
      v = d.one(ldf(sl.row + i));
      if (i == hit) v += extra;
    }
    stf(out + i, v);
  };
  if (!same) {
    for (int64_t i = sl.first(sl.v0) + t; i < sl.first(sl.v1); i += NT) one((int)i);
  } else if (zero) {
    for (int v = sl.v0 + t; v < sl.v1; v += NT)
      __stcs(reinterpret_cast<uint4 *>(out + sl.first(v)), make_uint4(0, 0, 0, 0));
  } else {
    // the vector of the element `hit`, counted in the calling thread's vectors, or -1
    int hv = -1;
    if (hit >= sl.first(sl.v0) && hit < sl.first(sl.v1)) {
      const int v = (int)(hit - sl.head) / N - sl.v0;
      if (v % NT == t) hv = v / NT;
    }
    uint4 *mine = ring_of<GW>(ring);
    const int last = ((sl.n + 1) >> 1) - 1;  // pair
    if (!KEPT) {
#pragma unroll
      for (int p = 0; p < RING; ++p) fetch_pair(sl, mine, last - p);
    }
    T *dst = out + sl.first(sl.v0 + t) + (int64_t)(2 * last) * sl.STEP;
    auto store = [&](const uint4 &raw, T *to, int i) {
      float x[N];
      Vec<T>::unpack(raw, x);
#pragma unroll
      for (int k = 0; k < N; k += 2) un2(d.two(f2(x[k], x[k + 1])), x[k], x[k + 1]);
      if (i == hv) {
        const int at = (int)(hit - sl.head) % N;
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k == at) x[k] += extra;
      }
      __stcs(reinterpret_cast<uint4 *>(to), Vec<T>::pack(x));
    };
    for (int p = last; p >= 0; --p) {
      copy_wait<RING - 1>();
      const uint4 *at = mine + (p % RING) * 2 * NT;
      store(at[0], dst, 2 * p);
      if (2 * p + 1 < sl.n) store(at[NT], dst + sl.STEP, 2 * p + 1);
      fetch_pair(sl, mine, p - RING);
      dst -= 2 * sl.STEP;
    }
  }
  if (t < sl.nhead) one(t);
  if (t < sl.ntail) one(sl.tail0 + t);
}

struct BwdArgs {
  const int64_t *targets;
  const float *stats, *entropy, *d_logprob, *d_entropy;
  float inv_t, c2;
  int V, shift;
  uint32_t rows;
};

// dx_j = (g (1{j = t} - p_j) - h p_j (log p_j + H)) / T
// HBM-bound: 8192 rows of 50280 bf16 logits, read once and written once, 261 us, 6.3 TB/s or 0.98 of the measured copy
// rate.
template <typename T, int GW, bool ENT>
__global__ void __launch_bounds__(CTA, GW == 1 ? 4 : 5) token_logprobs_bwd_kernel(const T *__restrict__ logits, Rows rows, BwdArgs a,
                                                                    T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  extern __shared__ uint4 ring[];
  const Part<GW> part(a.shift);
  if (GW == 1 && part.row >= a.rows) return;
  const int64_t r = part.row;
  const Slice<T, GW> sl(logits + rows.at(part.row), a.V, part.rank, part.shift);
  const float m = a.stats[2 * r], log_s = a.stats[2 * r + 1];
  const float h = ENT ? a.d_entropy[r] : 0.f;
  int64_t t = -1;
  float g = 0.f;
  if (a.d_logprob) {
    t = a.targets[r];
    g = t < 0 ? 0.f : t >= a.V ? NAN : a.d_logprob[r];
  }
  const float ent = ENT ? a.entropy[r] : 0.f;
  const bool zero = (g == 0.f && h == 0.f) || m == -INFINITY;
  const Dense<ENT> d(m, log_s, a.c2, -(g + h * ent) * a.inv_t, -h * LN2 * a.inv_t);
  write_grad<T, GW, false, ENT>(sl, grad + grows.at(part.row), d, zero, t, g * a.inv_t, ring);
}

// ----------------------------------------------------------------- distillation
struct DistillArgs {
  const int64_t *ids;
  const void *values;
  int v_dtype, k;
  const float *row_weight;
  float *loss, *stats;
  const float *stats_in;
  float inv_t, c2;
  int V, shift;
  uint32_t rows;
};

__device__ __forceinline__ float load_value(const void *p, int64_t i, int dtype) {
  return dtype == MTP_F32    ? ((const float *)p)[i]
         : dtype == MTP_BF16 ? __bfloat162float(((const __nv_bfloat16 *)p)[i])
                             : __half2float(((const __half *)p)[i]);
}

__device__ __forceinline__ float nan_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A row's teacher: token (-1: not used), probability, and the student's logit of entry i.
struct TeacherShared {
  alignas(16) int id[MAX_TOP];
  float q[MAX_TOP], x[MAX_TOP];
  float neg_entropy;  // sum q log q
  bool used, bad;     // any entry is used; a used one lies outside the vocabulary, or the probabilities are NaN
};

// By one warp, four entries a lane.
template <typename T>
__device__ __forceinline__ void read_teacher(const T *row, const DistillArgs &a, int64_t r, TeacherShared &te) {
  constexpr int PER = MAX_TOP / 32;
  const int lane = threadIdx.x & 31;
  int64_t id[PER];
  float t[PER], x[PER], m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane + 32 * j;
    id[j] = -1;
    t[j] = -INFINITY;
    if (i < a.k) {
      id[j] = a.ids[r * a.k + i];
      t[j] = load_value(a.values, r * a.k + i, a.v_dtype);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (id[j] < 0) t[j] = -INFINITY;
    x[j] = id[j] >= 0 && id[j] < a.V ? ldf(row + id[j]) : 0.f;
    m = nan_max(m, t[j]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = nan_max(m, __shfl_xor_sync(0xffffffffu, m, o));
  float e[PER], s = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    e[j] = t[j] == -INFINITY ? 0.f : expf((t[j] - m) * a.inv_t);
    s += e[j];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float ls = logf(s);
  bool bad = false;
  float neg = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane + 32 * j;
    const float q = s != 0.f ? e[j] / s : 0.f;
    bad = bad || q != q || (t[j] != -INFINITY && id[j] >= a.V);
    if (q != 0.f) neg += q * ((t[j] - m) * a.inv_t - ls);
    te.id[i] = q != 0.f && id[j] < a.V ? (int)id[j] : -1;
    te.q[i] = q;
    te.x[i] = x[j];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) neg += __shfl_xor_sync(0xffffffffu, neg, o);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    te.neg_entropy = neg;
    te.used = s != 0.f;
    te.bad = bad;
  }
}

// loss = sum q_i (log q_i - log p_id_i), dx_j = w (p_j - sum_{id_i = j} q_i) / T; q: softmax over the used entries of
// the teacher's logits / T.  GRAD: the gradient is written too.
// The teacher is read by one warp while the row streams in, and its elements of the gradient are written a second time
// by the CTA that wrote the row, after a barrier, so that the pass over the row does not look for them.
// Loss and gradient of 8192 rows of 50280 bf16 logits with 64 entries: 324 us against 256 us of HBM traffic (the second
// reading comes from shared memory and L2).  Bound by latency: nothing is loaded between a row's two passes (60% of the
// issue slots used, a warp's stalls are barriers and loads).  Keeping the whole slice in shared memory instead took
// clusters of two and 355 us.
template <typename T, int GW, bool GRAD>
__global__ void __launch_bounds__(CTA, GW == 1 ? 4 : 5) distill_kernel(const T *__restrict__ logits, Rows rows, DistillArgs a,
                                                         T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  using G = Group<GW>;
  extern __shared__ uint4 ring[];
  __shared__ RowShared sh;
  __shared__ TeacherShared teachers[G::ROWS];
  const Part<GW> part(a.shift);
  if (GW == 1 && part.row >= a.rows) return;
  TeacherShared &te = teachers[G::index()];
  const int parts = 1 << part.shift, rank = part.rank, t = G::tid();
  const int64_t r = part.row;
  const T *row = logits + rows.at(part.row);
  const Slice<T, GW> sl(row, a.V, rank, part.shift);
  const float w = GRAD ? a.row_weight[r] * a.inv_t : 0.f;
  RowStats st;
  if (a.stats_in) {
    if (t < 32) read_teacher(row, a, r, te);
    st = RowStats{a.stats_in[2 * r], a.stats_in[2 * r + 1], 0.f};
  } else {
    cluster_begin(parts);
    if (t < 32) read_teacher(row, a, r, te);
    const Stat own = thread_stats<T, GW, false, false>(sl, a.c2, ring, ChunkMaxima{});
    cluster_ready(parts);
    st = finish(row_join<GW, false>(own, sh, a.c2, rank, parts));
  }
  G::sync();
  if (rank == 0 && t < 32) {
    float loss = 0.f;
    for (int i = t; i < a.k; i += 32)
      if (te.q[i] != 0.f) loss -= te.q[i] * log_prob(te.x[i], st.m, st.log_s, a.inv_t);
#pragma unroll
    for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (t == 0) {
      if (a.loss) a.loss[r] = te.bad ? NAN : loss + te.neg_entropy;
      if (a.stats) {
        a.stats[2 * r] = st.m;
        a.stats[2 * r + 1] = st.log_s;
      }
    }
  }
  if constexpr (GRAD) {
    const bool zero = !te.used || w == 0.f || st.m == -INFINITY;
    T *out = grad + grows.at(part.row);
    const Dense<false> d(st.m, st.log_s, a.c2, te.bad ? NAN : w, 0.f);
    if (a.stats_in) write_grad<T, GW, false, false>(sl, out, d, zero, -1, 0.f, ring);
    else write_grad<T, GW, true, false>(sl, out, d, zero, -1, 0.f, ring);
    G::sync();  // the teacher's elements are written again, after the pass over all of them
    if (zero || te.bad) return;
    for (int i = t; i < a.k; i += G::NT) {
      const int id = te.id[i];
      const bool mine = id >= (rank == 0 ? 0 : sl.first(sl.v0)) && id < (rank == parts - 1 ? a.V : sl.first(sl.v1));
      if (!mine) continue;
      int same = 0;
      for (int j = 0; j < a.k; j += 4) {
        const int4 o = *reinterpret_cast<const int4 *>(te.id + j);
        same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
      }
      float qs = te.q[i];
      bool first = true;
      if (same > 1) {  // a token given more than once: the first entry of it writes the sum
        qs = 0.f;
        for (int j = 0; j < a.k; ++j) {
          if (te.id[j] != id) continue;
          first = first && j >= i;
          qs += te.q[j];
        }
      }
      if (first) stf(out + id, d.one(te.x[i]) - w * qs);
    }
  }
}

// How rows are shared out.  A warp takes a row of up to 16 KB where there are rows enough for 16 warps per SM: a CTA's
// fixed cost a row (its barriers and joins) is several times the work of such a row.  60000 rows of 1000 bf16 logits, loss
// and gradient with 64 entries: 126 us by warps (189 where tokens are given more than once), 474 by CTAs, against 37 of HBM
// traffic: the first load, the join and the stores of a row are a chain that only the SM's other warps overlap.  Else 2^shift
// CTAs share a row:
//   - until there is one for every SM, each with no fewer vectors than threads: a cluster adds about 2 us of barriers, so
//     more pays off only where SMs idle (64 rows of 50280 bf16 logits: 10.3 us by 4 CTAs, 12.3 by one; 300 rows: 18.4 by
//     2, 16.6 by one);
//   - where the row is read twice, until a CTA's part is at most TWICE bytes, so that what the CTAs at work read stays in
//     L2 (5 per SM x 104 KB = 77 MB of 126): 4096 rows of 50280 fp32 logits 338 us by 2 CTAs, 395 by one; 1024 of
//     131072 235 us by 8, 288 by one; 8192 of 50280 bf16 329 by one, 350 by two.
constexpr int64_t WARP_ROW = 16384, TWICE = 104 * 1024;
struct Share {
  bool warp;
  int shift;
  unsigned grid;
};
inline Share share_rows(int64_t rows, int V, int elem, bool twice, int top_k = 0) {
  const int64_t sms = num_sms(), bytes = (int64_t)V * elem;
  // for its alternatives a warp needs clearly more vectors than alternatives (60000 rows of 1000 bf16 logits, 125 vectors,
  // 128 alternatives: 1245 us by CTAs, 1671 by warps; 64 alternatives 264 by warps, 569 by CTAs, against 26 of HBM traffic)
  if (bytes <= WARP_ROW && rows >= 16 * sms && bytes / 16 >= top_k + top_k / 4)
    return {true, 0, (unsigned)((rows + Group<1>::ROWS - 1) / Group<1>::ROWS)};
  int shift = 0;
  while (2 << shift <= MAX_CLUSTER && bytes / 16 >> (shift + 1) >= CTA &&
         (rows << shift < sms || (twice && bytes >> shift > TWICE)))
    ++shift;
  return {false, shift, (unsigned)(rows << shift)};
}

// Launch with the CTAs of a row as a cluster.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_rows(void (*kern)(KArgs...), const Share &sh, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sh.grid);
  cfg.blockDim = dim3(CTA);
  cfg.dynamicSmemBytes = RING_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << sh.shift;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = sh.shift > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

template <typename T, int GW> auto fwd_kernel(bool ent, bool top) {
  return top ? (ent ? token_logprobs_kernel<T, GW, true, true> : token_logprobs_kernel<T, GW, false, true>)
             : (ent ? token_logprobs_kernel<T, GW, true, false> : token_logprobs_kernel<T, GW, false, false>);
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
  MTP_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "temperature must be between 1e-6 and 1e6");           \
  if (outer == 0 || inner == 0) return MTP_OK;                                                                    \
  MTP_REQUIRE(logits, "null pointer")

}  // namespace

// mtp_token_logprobs of arguments that have been checked.  expired: of fp32 logits, a word in device memory that is not 0 if
// they are not to be trusted (every log probability and entropy is then NaN); or null.
int launch_token_logprobs(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t ld_outer, int64_t ld, int V,
                          const int64_t *targets, float temperature, float *logprob, float *entropy, float *stats, int top_k,
                          int64_t *top_ids, float *top_logprobs, const int *expired, cudaStream_t stream) {
  const Rows rows = make_rows(outer, inner, ld_outer, ld);
  const int64_t n = outer * inner;
  const Share sh = share_rows(n, V, dtype == MTP_F32 ? 4 : 2, false, top_k);
  const FwdArgs a{targets, logprob, entropy, stats, top_k, top_ids, top_logprobs, 1.f / temperature,
                  (float)(1.4426950408889634 / temperature), V, sh.shift, (uint32_t)n, expired};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = sh.warp ? fwd_kernel<T, 1>(entropy, top_k > 0) : fwd_kernel<T, 8>(entropy, top_k > 0);
    launch_rows(kern, sh, stream, (const T *)logits, rows, a);
  });
  return check_launch("token_logprobs");
}

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
  return launch_token_logprobs(logits, dtype, outer, inner, ld_outer, ld, V, targets, temperature, logprob, entropy, stats,
                               top_k, top_ids, top_logprobs, nullptr, (cudaStream_t)stream);
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld), grows = make_rows(outer, inner, grad_ld_outer, grad_ld);
  const int64_t n = outer * inner;
  const Share sh = share_rows(n, V, dtype == MTP_F32 ? 4 : 2, false);
  const BwdArgs a{targets, stats, entropy, d_logprob, d_entropy, 1.f / temperature,
                  (float)(1.4426950408889634 / temperature), V, sh.shift, (uint32_t)n};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = sh.warp ? (d_entropy ? token_logprobs_bwd_kernel<T, 1, true> : token_logprobs_bwd_kernel<T, 1, false>)
                        : (d_entropy ? token_logprobs_bwd_kernel<T, 8, true> : token_logprobs_bwd_kernel<T, 8, false>);
    launch_rows(kern, sh, s, (const T *)logits, rows, a, (T *)grad, grows);
  });
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld);
  const int64_t n = outer * inner;
  const Share sh = share_rows(n, V, dtype == MTP_F32 ? 4 : 2, false);
  const DistillArgs a{ids, values, v_dtype, k, nullptr, loss, stats, nullptr, 1.f / temperature,
                      (float)(1.4426950408889634 / temperature), V, sh.shift, (uint32_t)n};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = sh.warp ? distill_kernel<T, 1, false> : distill_kernel<T, 8, false>;
    launch_rows(kern, sh, s, (const T *)logits, rows, a, (T *)nullptr, rows);
  });
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld), grows = make_rows(outer, inner, grad_ld_outer, grad_ld);
  const int64_t n = outer * inner;
  const Share sh = share_rows(n, V, dtype == MTP_F32 ? 4 : 2, stats == nullptr);
  const DistillArgs a{ids, values, v_dtype, k, row_weight, loss, nullptr, stats, 1.f / temperature,
                      (float)(1.4426950408889634 / temperature), V, sh.shift, (uint32_t)n};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = sh.warp ? distill_kernel<T, 1, true> : distill_kernel<T, 8, true>;
    launch_rows(kern, sh, s, (const T *)logits, rows, a, (T *)grad, grows);
  });
  return check_launch("distill_topk_grad");
}

}  // extern "C"

// Operators on logits rows: the log probability of a given token with entropy and top alternatives, its gradient, and
// the distillation loss from a teacher's top logits with its gradient.
//
// With z = x / T, m = max z and S = sum e^(z - m), a row gives
//   log p_j = (z_j - m) - log S          H = log S - sum e^(z - m) (z - m) / S
// All sums and statistics are fp32.  Every kernel reads a row in 16-byte vectors at the row's own alignment (the elements
// before the first and after the last whole vector one by one), a thread taking every 256th vector.  A forward pass
// reads its row once: each thread keeps the running maximum m, S and U = sum e^y y (y in units of log2) of its elements
// and rescales them when m grows; threads, and the CTAs of a cluster that share a row, are joined at the end.
#include <cooperative_groups.h>
#include "common.cuh"
#include "logits.cuh"

namespace mtp {
namespace {

namespace cg = cooperative_groups;
using namespace lg;

constexpr int MAX_TOP = 128;      // alternatives or teacher entries per row
constexpr int NT = 256;           // threads per CTA
constexpr int NW = NT / 32;
constexpr int MAX_CLUSTER = 8;    // CTAs that share a row
constexpr int LIST = 1024;        // candidates for the alternatives that a CTA holds

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

// CTA of a row: 2^shift of them share it.
struct Part {
  uint32_t row;
  int rank, shift;
  __device__ __forceinline__ explicit Part(int s) : row(blockIdx.x >> s), rank((int)(blockIdx.x & ((1u << s) - 1))), shift(s) {}
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
// row, the first CTA also the elements before them, the last the `tail` elements from `tail0` on.
template <typename T> struct Slice {
  const T *row;
  int head, v0, v1, nhead, tail0, ntail;
  __device__ __forceinline__ Slice(const T *r, int V, int rank, int shift) : row(r) {
    constexpr int N = Vec<T>::N;
    head = (int)(((16u - (unsigned)(reinterpret_cast<uintptr_t>(r) & 15u)) & 15u) / sizeof(T));
    if (head > V) head = V;
    const int nv = (V - head) / N;
    v0 = (int)((int64_t)nv * rank >> shift);
    v1 = (int)((int64_t)nv * (rank + 1) >> shift);
    nhead = rank == 0 ? head : 0;
    tail0 = head + nv * N;
    ntail = rank + 1 == 1 << shift ? V - tail0 : 0;
  }
  __device__ __forceinline__ const T *vec(int v) const { return row + head + (int64_t)v * Vec<T>::N; }
  __device__ __forceinline__ int first(int v) const { return head + v * Vec<T>::N; }  // index of a vector's first element
};

// ----------------------------------------------------------------- row statistics
// Asynchronous 16-byte copies into the calling thread's own places of shared memory: no thread reads another's, so that
// waiting for one's own copies is all the ordering that is needed.
__device__ __forceinline__ void copy16(uint4 *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// Vectors of the slice that thread t takes: v0 + t, v0 + t + NT, ...
template <typename T> __device__ __forceinline__ int thread_vectors(const Slice<T> &sl) {
  const int left = sl.v1 - sl.v0 - (int)threadIdx.x;
  return left > 0 ? (left + NT - 1) / NT : 0;
}

template <typename T, bool ENT>
__device__ __forceinline__ void accumulate_pair(Stat &st, const uint4 &a, const uint4 &b, float c2) {
  constexpr int N = Vec<T>::N;
  float x[2 * N], lo[N], hi[N];
  Vec<T>::unpack(a, lo);
  Vec<T>::unpack(b, hi);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = lo[i], x[N + i] = hi[i];
  accumulate<ENT, 2 * N>(st, x, c2);
}

template <typename T, bool ENT>
__device__ __forceinline__ void accumulate_vec(Stat &st, const uint4 &a, float c2) {
  constexpr int N = Vec<T>::N;
  float x[N];
  Vec<T>::unpack(a, x);
  accumulate<ENT, N>(st, x, c2);
}

template <typename T, bool ENT>
__device__ __forceinline__ void accumulate_ends(Stat &st, const Slice<T> &sl, float c2) {
  if (threadIdx.x < (unsigned)sl.nhead) accumulate1<ENT>(st, ldf(sl.row + threadIdx.x), c2);
  if (threadIdx.x < (unsigned)sl.ntail) accumulate1<ENT>(st, ldf(sl.row + sl.tail0 + threadIdx.x), c2);
}

// One thread's statistics of its elements, streamed through a ring of RING pairs of vectors per thread (32 KB a CTA, so
// that five CTAs keep 160 KB in flight on an SM whatever they compute).
constexpr int RING = 4, RING_BYTES = 2 * RING * NT * 16;
template <typename T, bool ENT>
__device__ __forceinline__ Stat thread_stats(const Slice<T> &sl, float c2, uint4 *ring) {
  Stat st{LOWEST, 0.f, 0.f};
  const int n = thread_vectors(sl);
  const T *src = sl.vec(sl.v0 + (int)threadIdx.x);
  constexpr int STEP = NT * Vec<T>::N;  // elements between a thread's vectors
  uint4 *mine = ring + threadIdx.x;
#pragma unroll
  for (int j = 0; j < RING; ++j) {
    if (2 * j < n) copy16(mine + (2 * j) * NT, src + (int64_t)(2 * j) * STEP);
    if (2 * j + 1 < n) copy16(mine + (2 * j + 1) * NT, src + (int64_t)(2 * j + 1) * STEP);
    copy_commit();
  }
  src += (int64_t)2 * RING * STEP;
  int slot = 0;
  for (int i = 0; i < n; i += 2) {
    copy_wait<RING - 1>();
    uint4 *at = mine + slot * 2 * NT;
    if (i + 1 < n) accumulate_pair<T, ENT>(st, at[0], at[NT], c2);
    else accumulate_vec<T, ENT>(st, at[0], c2);
    if (i + 2 * RING < n) copy16(at, src);
    if (i + 2 * RING + 1 < n) copy16(at + NT, src + STEP);
    copy_commit();
    src += 2 * STEP;
    slot = (slot + 1) & (RING - 1);
  }
  accumulate_ends<T, ENT>(st, sl, c2);
  return st;
}

// The same with the whole slice kept in shared memory, at most RESIDENT vectors per thread, all of them in flight at once.
constexpr int RESIDENT = 13, RESIDENT_BYTES = RESIDENT * NT * 16;
template <typename T> __device__ __forceinline__ void resident_fetch(const Slice<T> &sl, uint4 *keep) {
  const int n = thread_vectors(sl);
  const T *src = sl.vec(sl.v0 + (int)threadIdx.x);
  constexpr int STEP = NT * Vec<T>::N, PAIRS = (RESIDENT + 1) / 2;
  uint4 *mine = keep + threadIdx.x;
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    if (2 * j < n) copy16(mine + (2 * j) * NT, src + (int64_t)(2 * j) * STEP);
    if (2 * j + 1 < n) copy16(mine + (2 * j + 1) * NT, src + (int64_t)(2 * j + 1) * STEP);
    copy_commit();
  }
}

template <typename T, bool ENT>
__device__ __forceinline__ Stat resident_stats(const Slice<T> &sl, float c2, const uint4 *keep) {
  Stat st{LOWEST, 0.f, 0.f};
  const int n = thread_vectors(sl);
  const uint4 *mine = keep + threadIdx.x;
  constexpr int PAIRS = (RESIDENT + 1) / 2;
  auto step = [&](int j) {
    if (2 * j + 1 < n) accumulate_pair<T, ENT>(st, mine[2 * j * NT], mine[(2 * j + 1) * NT], c2);
    else if (2 * j < n) accumulate_vec<T, ENT>(st, mine[2 * j * NT], c2);
  };
  static_assert(PAIRS == 7, "one wait per pair below");
  copy_wait<6>(); step(0);
  copy_wait<5>(); step(1);
  copy_wait<4>(); step(2);
  copy_wait<3>(); step(3);
  copy_wait<2>(); step(4);
  copy_wait<1>(); step(5);
  copy_wait<0>(); step(6);
  accumulate_ends<T, ENT>(st, sl, c2);
  return st;
}

// Shared state of the CTAs of a row.  Every CTA gets every CTA's statistics (and group maxima) in its own copy.
struct RowShared {
  float m[NW];
  float2 su[NW];
  Stat cta[MAX_CLUSTER];
};

// Joins the threads of the CTA and the CTAs of the cluster; every thread of the cluster returns the row's statistics.
// The CTA's maximum comes first, so that each thread rescales its sums once and the rest are additions, in an order
// that is the same in every thread.  Orders the shared memory written before it (the group maxima, peers' copies
// included) for all threads.
// cluster_begin, called once before: a CTA of the cluster says that it runs and its shared memory may be written.
__device__ __forceinline__ void cluster_begin(int parts) {
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_ready(int parts) {
  if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

template <bool ENT>
__device__ __forceinline__ Stat row_join(Stat st, RowShared &sh, float c2, int rank, int parts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(st.m));
  if (lane == 0) sh.m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) m = fmaxf(m, sh.m[i]);
  const float y = fmaxf((st.m - m) * c2, FLOOR_Y), e = ex2(y);
  float u = ENT ? fmaf(y, st.s, st.u) * e : 0.f, s = st.s * e;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    if (ENT) u += __shfl_xor_sync(0xffffffffu, u, o);
  }
  if (lane == 0) sh.su[warp] = make_float2(s, u);
  __syncthreads();
  Stat all{m, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NW; ++i) {
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
  return all;
}

template <typename F, typename T>
__device__ __forceinline__ T block_reduce(T v, T *red, F op) {
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  T s = red[0];
  for (int i = 1; i < NW; ++i) s = op(s, red[i]);  // fixed order: the same in every thread
  return s;
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

// The k largest of a row without a second pass over it.  The threads of all CTAs form NT groups (a group is `parts`
// neighbouring threads of a CTA); the k-th largest of the groups' maxima is a lower bound of the row's k-th largest
// element, since each of k groups holds an element that is not below it.  Only threads whose own maximum reaches the
// bound look at their elements again (k = 64 of 50280: about 75 threads) and put those that reach it on the CTA's
// list.  The lists of the cluster are joined in its first CTA, and an element's place in the result is the number of
// elements above it.
struct TopShared {
  uint32_t group[NT];   // order keys of the groups' maxima, all CTAs'
  uint64_t *list;       // [LIST] this CTA's candidates, [MAX_CLUSTER * MAX_TOP] the cluster's after them: both lie in
                        // the ring, which has been read when the first candidate is written
  uint64_t red[NW];
  unsigned char lanes[NW][32];
  uint32_t bound;
  int n;
};

// Largest b with at least k of the NT keys >= b, or a smaller one that fewer than k + k / 8 + 4 reach.  One warp.
__device__ __forceinline__ uint32_t group_bound(const uint32_t *group, int k) {
  const int lane = threadIdx.x & 31;
  uint32_t key[NW], lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    key[i] = group[lane + 32 * i];
    lo = min(lo, key[i]);
    hi = max(hi, key[i]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  const int enough = k + k / 8 + 4;
  // all NT >= k keys reach lo; fewer than k, or nobody knows yet, reach more than hi
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    int c = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) c += key[i] >= mid;
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

// Calls f(value, index) for the elements of those threads of the calling warp whose bit in `todo` is set.  The lanes
// share all of their vectors, four loads in flight each.  lanes: 32 bytes of shared memory of the warp.
template <typename T, typename F>
__device__ __forceinline__ void warp_elements(const Slice<T> &sl, unsigned todo, unsigned char *lanes, F f) {
  constexpr int N = Vec<T>::N, DEPTH = 4;
  const int lane = threadIdx.x & 31, warp0 = threadIdx.x & ~31;
  if (todo >> lane & 1) lanes[__popc(todo & ((1u << lane) - 1))] = (unsigned char)lane;
  __syncwarp();
  const int each = (sl.v1 - sl.v0 + NT - 1) / NT, items = __popc(todo) * each;
  for (int base = 0; base < items; base += 32 * DEPTH) {
    uint4 raw[DEPTH];
    int at[DEPTH];
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const int item = base + 32 * j + lane;
      at[j] = -1;
      if (item < items) {
        const int v = sl.v0 + warp0 + lanes[item / each] + (item % each) * NT;
        if (v < sl.v1) {
          at[j] = sl.first(v);
          raw[j] = load16(sl.vec(v));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      if (at[j] >= 0) {
        float x[N];
        Vec<T>::unpack(raw[j], x);
#pragma unroll
        for (int i = 0; i < N; ++i) f(x[i], at[j] + i);
      }
    }
  }
  if (todo >> lane & 1) {
    const int t = threadIdx.x;
    if (t < sl.nhead) f(ldf(sl.row + t), t);
    if (t < sl.ntail) f(ldf(sl.row + sl.tail0 + t), sl.tail0 + t);
  }
}

// The same for a thread's own elements.
template <typename T, typename F>
__device__ __forceinline__ void thread_elements(const Slice<T> &sl, F f) {
  constexpr int N = Vec<T>::N;
  const int t = threadIdx.x;
  for (int v = sl.v0 + t; v < sl.v1; v += NT) {
    float x[N];
    Vec<T>::unpack(load16(sl.vec(v)), x);
#pragma unroll
    for (int i = 0; i < N; ++i) f(x[i], sl.first(v) + i);
  }
  if (t < sl.nhead) f(ldf(sl.row + t), t);
  if (t < sl.ntail) f(ldf(sl.row + sl.tail0 + t), sl.tail0 + t);
}

__device__ __forceinline__ uint64_t count_op(uint64_t a, uint64_t b) { return a + b; }

// Largest key that at least k of the counted elements reach, or a smaller one that at most `most` >= k reach.
// count(key): how many elements of the calling thread are >= key; lo: a key that at least k reach; no key is above hi.
template <typename F>
__device__ uint64_t key_bound(uint64_t lo, uint64_t hi, int k, int most, uint64_t *red, F count) {
  auto add = [](uint64_t a, uint64_t b) { return count_op(a, b); };
  while (lo < hi) {
    const uint64_t mid = lo + (hi - lo) / 2 + 1;
    const uint64_t c = block_reduce((uint64_t)count(mid), red, add);
    if (c >= (uint64_t)k) {
      lo = mid;
      if (c <= (uint64_t)most) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// Cuts list[0, n) down to at most `most` >= k keys, the k largest among them; n <= LIST.
__device__ int cut_list(uint64_t *list, int n, int k, int most, TopShared &sh) {
  if (n <= most) return n;
  const uint64_t b = key_bound(0, ~0ull, k, most, sh.red, [&](uint64_t key) {
    int c = 0;
    for (int i = threadIdx.x; i < n; i += NT) c += list[i] >= key;
    return c;
  });
  uint64_t mine[LIST / NT];
#pragma unroll
  for (int i = 0; i < LIST / NT; ++i) {
    const int at = threadIdx.x + i * NT;
    mine[i] = at < n ? list[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < LIST / NT; ++i)
    if (mine[i] >= b && threadIdx.x + i * NT < n) list[atomicAdd(&sh.n, 1)] = mine[i];
  __syncthreads();
  return sh.n;
}

// st: the calling thread's own statistics, total: the row's; group maxima are in place (row_join has ordered them).
template <typename T>
__device__ void top_alternatives(const Slice<T> &sl, Stat st, RowStats row, int k, float inv_t, int V, TopShared &sh,
                                 int rank, int parts, int64_t *ids, float *logprobs) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const uint32_t b = group_bound(sh.group, k);
    if (lane == 0) {
      sh.bound = b;
      sh.n = 0;
    }
  }
  __syncthreads();
  const uint32_t bound = sh.bound;
  // a thread whose sum is NaN may hold a NaN, which its maximum passes over
  const unsigned todo =
      __ballot_sync(0xffffffffu, order_key(st.s == 0.f ? -INFINITY : st.m) >= bound || st.s != st.s);
  const float least = key_value(bound);  // bound 0 (a group without an element) gives NaN, which everything passes
  warp_elements(sl, todo, sh.lanes[warp], [&](float x, int i) {
    if (!(x < least)) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < LIST) sh.list[at] = element_key(x, i);
    }
  });
  __syncthreads();
  int n = sh.n;
  if (n > LIST) {
    // more elements reach the bound than the list holds (a row of equal logits): find the key of this CTA's k-th
    // largest element by bisection, one scan of the slice a step, and collect again
    const uint64_t lo = ((uint64_t)bound << 32) | (uint32_t)~(V - 1);
    const uint64_t hi = row.log_s != row.log_s ? ~0ull : ((uint64_t)order_key(row.m) << 32) | 0xFFFFFFFFu;
    const uint64_t b = key_bound(lo, hi, k, MAX_TOP, sh.red, [&](uint64_t key) {
      int c = 0;
      thread_elements(sl, [&](float x, int i) { c += element_key(x, i) >= key; });
      return c;
    });
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    thread_elements(sl, [&](float x, int i) {
      const uint64_t key = element_key(x, i);
      if (key >= b) sh.list[atomicAdd(&sh.n, 1)] = key;
    });
    __syncthreads();
    n = sh.n;
  }
  const uint64_t *list = sh.list;
  if (parts > 1) {
    n = cut_list(sh.list, n, k, MAX_TOP, sh);
    __syncthreads();
    if (threadIdx.x == 0) sh.n = n;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (rank == 0) {
      int at = 0;
      for (int c = 0; c < parts; ++c) {
        const int nc = *cl.map_shared_rank(&sh.n, c);
        const uint64_t *from = cl.map_shared_rank(sh.list, c);
        if (threadIdx.x < (unsigned)nc) sh.list[LIST + at + threadIdx.x] = from[threadIdx.x];
        at += nc;
      }
      n = at;
    }
    cl.sync();  // the peers' lists have been read
    if (rank != 0) return;
    list = sh.list + LIST;
  }
  n = cut_list(const_cast<uint64_t *>(list), n, k, NT, sh);
  if (threadIdx.x < (unsigned)n) {
    const uint64_t key = list[threadIdx.x];
    int place = 0;
    for (int i = 0; i < n; ++i) place += list[i] > key;
    if (place < k) {
      ids[place] = (int64_t)(int)~(uint32_t)key;
      logprobs[place] = log_prob(key_value((uint32_t)(key >> 32)), row.m, row.log_s, inv_t);
    }
  }
}

// ----------------------------------------------------------------- log probabilities
struct FwdArgs {
  const int64_t *targets;
  float *logprob, *entropy, *stats;
  int top_k;
  int64_t *top_ids;
  float *top_logprobs;
  float inv_t, c2;  // 1 / T, log2 e / T
  int V, shift;
};

template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(NT, 5) token_logprobs_kernel(const T *__restrict__ logits, Rows rows, FwdArgs a) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  __shared__ RowShared sh;
  __shared__ TopShared top;
  __shared__ uint4 ring[2 * RING * NT];
  static_assert(sizeof(ring) >= 8 * (LIST + MAX_CLUSTER * MAX_TOP), "the ring holds the lists");
  const Part part(a.shift);
  const int parts = 1 << a.shift, rank = part.rank;
  const int64_t r = part.row;
  const T *row = logits + rows.at(part.row);
  const Slice<T> sl(row, a.V, rank, a.shift);
  cluster_begin(parts);
  const Stat st = thread_stats<T, ENT>(sl, a.c2, ring);
  cluster_ready(parts);
  if constexpr (TOP) {
    if (threadIdx.x == 0) top.list = reinterpret_cast<uint64_t *>(ring);
    // maxima of groups of `parts` threads to every CTA of the cluster
    uint32_t g = sl.v0 + (int)threadIdx.x < sl.v1 || threadIdx.x < (unsigned)sl.nhead || threadIdx.x < (unsigned)sl.ntail
                     ? order_key(st.s == 0.f ? -INFINITY : st.m)
                     : 0u;
    for (int o = 1; o < parts; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    const int slot = rank * (NT >> a.shift) + ((int)threadIdx.x >> a.shift);
    const int to = threadIdx.x & (parts - 1);
    if (parts > 1) *cg::this_cluster().map_shared_rank(&top.group[slot], to) = g;
    else top.group[slot] = g;
  }
  const Stat all = row_join<ENT>(st, sh, a.c2, rank, parts);
  if (!TOP && threadIdx.x >= 32) return;
  const RowStats s = finish(all);
  if (rank == 0 && threadIdx.x == 0) {
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
    top_alternatives(sl, st, s, a.top_k, a.inv_t, a.V, top, rank, parts, a.top_ids + r * a.top_k,
                     a.top_logprobs + r * a.top_k);
}

// ----------------------------------------------------------------- gradients
// out_j = p_j (a + b y_j) with p_j = 2^y_j, y = log2 p; the element `hit` gets `extra` on top.  ENT: b is not 0.
// A p below 2^-126 still counts where its factor is large: 2^(y + 32) is taken, which is flushed to zero only where p
// is below the smallest subnormal, and 2^-32 goes into the factor.
template <bool ENT> struct Dense {
  float m, l2, c2;  // largest logit, log2 S, log2 e / T
  float a, b;       // times 2^-32
  static constexpr float LIFT = 32.f;
  __device__ __forceinline__ Dense(float m_, float log_s, float c2_, float a_, float b_)
      : m(m_), l2(log_s * LOG2E), c2(c2_), a(a_ * 0x1p-32f), b(b_ * 0x1p-32f) {
    if (!ENT) l2 -= LIFT;
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
      un2(add2(y, f2(LIFT, LIFT)), y0, y1);
      return mul2(f2(ex2(y0), ex2(y1)), f);
    }
  }
  __device__ __forceinline__ float one(float x) const {
    float v, w;
    un2(two(f2(x, x)), v, w);
    return v;
  }
};

// Writes the slice's gradient.  16-byte stores where the gradient row is aligned as the logits row is.  KEPT: the vectors
// are where resident_stats left them in shared memory.
template <typename T, bool KEPT, bool ENT>
__device__ __forceinline__ void write_grad(const Slice<T> &sl, T *out, const Dense<ENT> &d, bool zero, int64_t hit,
                                           float extra, const uint4 *kept) {
  constexpr int N = Vec<T>::N, DEPTH = 4;
  const bool same = ((reinterpret_cast<uintptr_t>(sl.row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  auto one = [&](int i) {
    float v = 0.f;
    if (!zero) {
      v = d.one(ldf(sl.row + i));
      if (i == hit) v += extra;
    }
    stf(out + i, v);
  };
  if (!same) {
    for (int64_t i = sl.first(sl.v0) + (int)threadIdx.x; i < sl.first(sl.v1); i += NT) one((int)i);
  } else if (zero) {
    for (int v = sl.v0 + threadIdx.x; v < sl.v1; v += NT)
      __stcs(reinterpret_cast<uint4 *>(out + sl.first(v)), make_uint4(0, 0, 0, 0));
  } else {
    const int n = thread_vectors(sl), v0 = sl.v0 + (int)threadIdx.x;
    const int hv = hit >= sl.first(sl.v0) && hit < sl.first(sl.v1) ? (int)((hit - sl.head) / N) : -1;
    const T *src = sl.vec(v0);
    T *dst = out + sl.first(v0);
    const uint4 *keep = kept + threadIdx.x;
    constexpr int STEP = NT * N;
    for (int i = 0; i < n; i += DEPTH) {
      uint4 raw[DEPTH];
#pragma unroll
      for (int j = 0; j < DEPTH; ++j)
        if (i + j < n) raw[j] = KEPT ? keep[(i + j) * NT] : load16(src + j * STEP);
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        if (i + j < n) {
          float x[N];
          Vec<T>::unpack(raw[j], x);
#pragma unroll
          for (int k = 0; k < N; k += 2) un2(d.two(f2(x[k], x[k + 1])), x[k], x[k + 1]);
          if (v0 + (i + j) * NT == hv) {
            const int at = (int)(hit - sl.first(hv));
#pragma unroll
            for (int k = 0; k < N; ++k)
              if (k == at) x[k] += extra;
          }
          __stcs(reinterpret_cast<uint4 *>(dst + j * STEP), Vec<T>::pack(x));
        }
      }
      src += DEPTH * STEP;
      dst += DEPTH * STEP;
    }
  }
  if (threadIdx.x < (unsigned)sl.nhead) one(threadIdx.x);
  if (threadIdx.x < (unsigned)sl.ntail) one(sl.tail0 + threadIdx.x);
}

struct BwdArgs {
  const int64_t *targets;
  const float *stats, *entropy, *d_logprob, *d_entropy;
  float inv_t, c2;
  int V, shift;
};

// dx_j = (g (1{j = t} - p_j) - h p_j (log p_j + H)) / T
template <typename T, bool ENT>
__global__ void __launch_bounds__(NT, 4) token_logprobs_bwd_kernel(const T *__restrict__ logits, Rows rows, BwdArgs a,
                                                                   T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  const Part part(a.shift);
  const int64_t r = part.row;
  const Slice<T> sl(logits + rows.at(part.row), a.V, part.rank, a.shift);
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
  write_grad<T, false, ENT>(sl, grad + grows.at(part.row), d, zero, t, g * a.inv_t, nullptr);
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

// A row's teacher: token, probability, its log, and the student's logit of entry i; entries that are not used have q = 0.
struct TeacherShared {
  int64_t id[MAX_TOP];
  float q[MAX_TOP], log_q[MAX_TOP], x[MAX_TOP];
  bool used, bad;  // any entry is used; a used one lies outside the vocabulary, or the probabilities are NaN
};

// By one warp, four entries a lane.
template <typename T>
__device__ __forceinline__ void read_teacher(const T *row, const DistillArgs &a, int64_t r, TeacherShared &te) {
  constexpr int PER = MAX_TOP / 32;
  const int lane = threadIdx.x;
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
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane + 32 * j;
    const float q = s != 0.f ? e[j] / s : 0.f;
    bad = bad || q != q || (q != 0.f && id[j] >= a.V);
    if (i < a.k) {
      te.id[i] = id[j];
      te.q[i] = q;
      te.log_q[i] = (t[j] - m) * a.inv_t - ls;
      te.x[i] = x[j];
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    te.used = s != 0.f;
    te.bad = bad;
  }
}

// loss = sum q_i (log q_i - log p_id_i), dx_j = w (p_j - sum_{id_i = j} q_i) / T; q: softmax over the used entries of
// the teacher's logits / T, thread i holding entry i.  GRAD: the gradient is written too.  RES: the slice stays in shared
// memory between the statistics and the gradient, so that the logits are read from memory once.
template <typename T, bool GRAD, bool RES>
__global__ void __launch_bounds__(NT, GRAD ? 4 : 5) distill_kernel(const T *__restrict__ logits, Rows rows, DistillArgs a,
                                                        T *__restrict__ grad, Rows grows) {
  MTP_PDL_WAIT();
  MTP_PDL_TRIGGER();
  extern __shared__ uint4 buffer[];  // the ring, or with RES the slice
  __shared__ RowShared sh;
  __shared__ TeacherShared te;
  const Part part(a.shift);
  const int parts = 1 << a.shift, rank = part.rank;
  const int64_t r = part.row;
  const T *row = logits + rows.at(part.row);
  const Slice<T> sl(row, a.V, rank, a.shift);
  const float w = GRAD ? a.row_weight[r] * a.inv_t : 0.f;
  if (!a.stats_in) cluster_begin(parts);
  if (RES) resident_fetch(sl, buffer);
  if (threadIdx.x < 32) read_teacher(row, a, r, te);  // while the slice is on its way
  RowStats st;
  if (a.stats_in) {
    st = RowStats{a.stats_in[2 * r], a.stats_in[2 * r + 1], 0.f};
    __syncthreads();
  } else {
    const Stat own = RES ? resident_stats<T, false>(sl, a.c2, buffer) : thread_stats<T, false>(sl, a.c2, buffer);
    cluster_ready(parts);
    st = finish(row_join<false>(own, sh, a.c2, rank, parts));
  }
  if (rank == 0 && threadIdx.x < 32) {
    float loss = 0.f;
    for (int i = threadIdx.x; i < a.k; i += 32)
      if (te.q[i] != 0.f) loss += te.q[i] * (te.log_q[i] - log_prob(te.x[i], st.m, st.log_s, a.inv_t));
#pragma unroll
    for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
    if (threadIdx.x == 0) {
      if (a.loss) a.loss[r] = te.bad ? NAN : loss;
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
    write_grad<T, RES, false>(sl, out, d, zero, -1, 0.f, buffer);
    __syncthreads();  // the teacher's elements are written again, after the pass over all of them
    if (threadIdx.x >= (unsigned)a.k || zero || te.bad) return;
    const int64_t id = te.id[threadIdx.x];
    const bool mine = id >= (rank == 0 ? 0 : sl.first(sl.v0)) && id < (rank == parts - 1 ? a.V : sl.first(sl.v1));
    if (te.q[threadIdx.x] != 0.f && mine) {
      float qs = 0.f;
      bool first = true;
      for (int j = 0; j < a.k; ++j) {
        if (te.id[j] == id) {
          qs += te.q[j];
          first = first && (j >= (int)threadIdx.x || te.q[j] == 0.f);
        }
      }
      const float lp = log_prob(te.x[threadIdx.x], st.m, st.log_s, a.inv_t);
      if (first) stf(out + id, w * (ex2(lp * LOG2E) - qs));
    }
  }
}

// log2 of the CTAs that share a row: rows alone fill the GPU from about four CTAs per SM on; a CTA takes no fewer than NT
// vectors.
inline int row_shift(int64_t rows, int V, int elem) {
  const int64_t want = 4ll * num_sms();
  const int64_t vecs = (int64_t)V * elem / 16;
  int shift = 0;
  while (2 << shift <= MAX_CLUSTER && rows << shift < want && vecs >> (shift + 1) >= NT) ++shift;
  return shift;
}

// Launch with the CTAs of a row as a cluster.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_rows(void (*kern)(KArgs...), int64_t rows, int shift, size_t smem, cudaStream_t stream,
                               Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows << shift));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << shift;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = shift > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld);
  const int64_t n = outer * inner;
  const int shift = row_shift(n, V, dtype == MTP_F32 ? 4 : 2);
  const FwdArgs a{targets, logprob, entropy, stats, top_k, top_ids, top_logprobs, 1.f / temperature,
                  (float)(1.4426950408889634 / temperature), V, shift};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = top_k ? (entropy ? token_logprobs_kernel<T, true, true> : token_logprobs_kernel<T, false, true>)
                      : (entropy ? token_logprobs_kernel<T, true, false> : token_logprobs_kernel<T, false, false>);
    launch_rows(kern, n, shift, 0, s, (const T *)logits, rows, a);
  });
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld), grows = make_rows(outer, inner, grad_ld_outer, grad_ld);
  const int64_t n = outer * inner;
  const int shift = row_shift(n, V, dtype == MTP_F32 ? 4 : 2);
  const BwdArgs a{targets, stats, entropy, d_logprob, d_entropy, 1.f / temperature,
                  (float)(1.4426950408889634 / temperature), V, shift};
  MTP_DISPATCH_LOGITS(dtype, T, {
    auto kern = d_entropy ? token_logprobs_bwd_kernel<T, true> : token_logprobs_bwd_kernel<T, false>;
    launch_pdl(kern, dim3((unsigned)(n << shift)), dim3(NT), 0, s, (const T *)logits, rows, a, (T *)grad, grows);
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
  const int shift = row_shift(n, V, dtype == MTP_F32 ? 4 : 2);
  const DistillArgs a{ids, values, v_dtype, k, nullptr, loss, stats, nullptr, 1.f / temperature,
                      (float)(1.4426950408889634 / temperature), V, shift};
  MTP_DISPATCH_LOGITS(dtype, T, launch_rows(distill_kernel<T, false, false>, n, shift, RING_BYTES, s,
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
  const Rows rows = make_rows(outer, inner, ld_outer, ld), grows = make_rows(outer, inner, grad_ld_outer, grad_ld);
  const int64_t n = outer * inner;
  const int elem = dtype == MTP_F32 ? 4 : 2;
  int shift = row_shift(n, V, elem);
  // keep the slices resident: more CTAs per row until a slice fits
  auto fits = [&](int c) { return (((int64_t)V * elem / 16 - 1) >> c) + 1 <= RESIDENT * NT; };
  bool res = stats == nullptr;
  if (res) {
    int c = shift;
    while (2 << c <= MAX_CLUSTER && !fits(c)) ++c;
    res = fits(c);
    if (res) shift = c;
  }
  const DistillArgs a{ids, values, v_dtype, k, row_weight, loss, nullptr, stats, 1.f / temperature,
                      (float)(1.4426950408889634 / temperature), V, shift};
  MTP_DISPATCH_LOGITS(dtype, T, {
    if (res) {
      // set at every call: the attribute belongs to the current device
      if (cudaFuncSetAttribute(distill_kernel<T, true, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               RESIDENT_BYTES) != cudaSuccess)
        return fail(MTP_ERR_CUDA, "distill_topk_grad: shared memory");
      launch_rows(distill_kernel<T, true, true>, n, shift, RESIDENT_BYTES, s, (const T *)logits, rows, a, (T *)grad, grows);
    } else {
      launch_rows(distill_kernel<T, true, false>, n, shift, RING_BYTES, s, (const T *)logits, rows, a, (T *)grad, grows);
    }
  });
  return check_launch("distill_topk_grad");
}

}  // extern "C"

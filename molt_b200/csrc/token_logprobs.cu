// Log-probabilities of given tokens from logits, and their gradient with respect to the logits.
//   l = (x_t - M) / T - ln S,   S = sum_v exp((x_v - M) / T),   dl/dx_v = (1[v = t] - p_v) / T,   p_v = exp((x_v - M) / T) / S
// Everything is computed from differences x - M, which are exact or nearly so: the rounding of log2(e) / T then changes l
// only by a relative 2^-24 of such a difference, and logits at the type's lowest value neither overflow nor make NaN.
#include <math.h>

#include "common.cuh"

namespace molt {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float exp2_fast(float v) {   // 2^-22 relative
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Pairs of fp32 in one 64-bit register: one instruction for two additions, products or fused products.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair(float a, float b) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(pair_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
  pair_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t exp2_2(pair_t v) {
  const float2 h = halves(v);
  return pair(exp2_fast(h.x), exp2_fast(h.y));
}

// What the kernels need of 16 bytes of logits.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kElements = 4;
  static __device__ __forceinline__ float largest(const uint4& q, float m) {
    return fmaxf(fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w))), m);
  }
  // f of every pair of differences x - m
  template <typename F>
  static __device__ __forceinline__ void each(const uint4& q, float m, F f) {
    const pair_t minus = pair(-m, -m);
    f(add2(pair(__uint_as_float(q.x), __uint_as_float(q.y)), minus));
    f(add2(pair(__uint_as_float(q.z), __uint_as_float(q.w)), minus));
  }
  template <typename F>
  static __device__ __forceinline__ uint4 map(const uint4& q, float m, F f) {
    const pair_t minus = pair(-m, -m);
    const float2 a = halves(f(add2(pair(__uint_as_float(q.x), __uint_as_float(q.y)), minus)));
    const float2 b = halves(f(add2(pair(__uint_as_float(q.z), __uint_as_float(q.w)), minus)));
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kElements = 8;
  static __device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {   // drops a NaN, which the sum then carries
    unsigned r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float largest(const uint4& q, float m) {
    const unsigned v = max2(max2(q.x, q.y), max2(q.z, q.w));
    return fmaxf(m, fmaxf(bf16_lo(v), bf16_hi(v)));
  }
  // x - m in fp32 straight from the bf16 halves of a word, one instruction each
  static __device__ __forceinline__ pair_t differences(unsigned w, float m) {
    float a, b;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tsub.rn.f32.bf16 %0, lo, %3;\n\tsub.rn.f32.bf16 %1, hi, %3;\n\t}"
        : "=f"(a), "=f"(b) : "r"(w), "f"(m));
    return pair(a, b);
  }
  template <typename F>
  static __device__ __forceinline__ void each(const uint4& q, float m, F f) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f(differences(w[i], m));
  }
  template <typename F>
  static __device__ __forceinline__ uint4 map(const uint4& q, float m, F f) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    unsigned o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = halves(f(differences(w[i], m)));
      o[i] = pack_bf16x2(h.x, h.y);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
};

// ---- the running pair (maximum m, sum s of exp2((x - m) c)) -----------------------------------------------------------
// A part without a finite logit has m = -inf and s = 0; a NaN logit leaves NaN in s; m = +inf makes inf - inf in s.
struct Running {
  float m = -INFINITY;
  pair_t s = 0;   // two partial sums
  float c;

  // What the exponents are taken from: -inf - -inf must not arise while only -inf has been seen.
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void raise(float to) {
    const float before = m;
    m = to;
    const float k = exp2_fast((before - base()) * c);
    s = mul2(s, pair(k, k));
  }
  template <typename T, int N>
  __device__ __forceinline__ void take(const uint4 (&q)[N]) {
    float top = m;
#pragma unroll
    for (int j = 0; j < N; ++j) top = Vec<T>::largest(q[j], top);
    raise(top);
    const float from = base();
    const pair_t cc = pair(c, c);
#pragma unroll
    for (int j = 0; j < N; ++j) Vec<T>::each(q[j], from, [&](pair_t d) { s = add2(s, exp2_2(mul2(d, cc))); });
  }
  // The same with a reference that stays until a batch exceeds it by 2^8: sums stay far from fp32's limits, ln s (whose
  // rounding stays in the result) stays small, and the rescaling is hardly ever executed.
  template <typename T, int N>
  __device__ __forceinline__ void take_lazily(const uint4 (&q)[N]) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) top = Vec<T>::largest(q[j], top);
    if (top > m + 8.f / c) raise(top);
    const float from = base();
    const pair_t cc = pair(c, c);
#pragma unroll
    for (int j = 0; j < N; ++j) Vec<T>::each(q[j], from, [&](pair_t d) { s = add2(s, exp2_2(mul2(d, cc))); });
  }
  __device__ __forceinline__ void take_one(float x) {
    raise(fmaxf(m, x));
    s = add2(s, pair(exp2_fast((x - base()) * c), 0.f));
  }
};

__device__ __forceinline__ void warp_join(float& m, float& s, float c) {
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  s = m == top ? s : s * exp2_fast((m - top) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  m = top;
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_in_cta(float2* slot, unsigned cta, float2 v) {
  const unsigned local = (unsigned)__cvta_generic_to_shared(slot);
  unsigned remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(cta));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}

// Joins the pairs of all threads that share a row; every thread gets the result.  The caller's cluster has arrived at the
// cluster barrier once (so that every block's shared memory exists before another block writes to it).
template <int THREADS>
__device__ __forceinline__ void row_join(float& m, float& s, float c, unsigned rank, unsigned size) {
  __shared__ float2 of_warp[32], of_cta[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  warp_join(m, s, c);
  if (lane == 0) of_warp[warp] = make_float2(m, s);
  __syncthreads();
  float2 q = lane < THREADS / 32 ? of_warp[lane] : make_float2(-INFINITY, 0.f);
  m = q.x;
  s = q.y;
  warp_join(m, s, c);
  if (size > 1) {
    cluster_wait();
    if (warp == 0 && lane < size) store_in_cta(of_cta + rank, lane, make_float2(m, s));
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    q = lane < size ? of_cta[lane] : make_float2(-INFINITY, 0.f);
    m = q.x;
    s = q.y;
    warp_join(m, s, c);
  }
}

// Where the rows of logits lie: `group` rows (0: all of them) one `stride` apart, then the next group.  Two strides are what
// logits[:, :-1] needs to be read where it is; the division is one per block.
struct Layout {
  long long stride, group_stride;
  unsigned group;
  __device__ __forceinline__ long long of(unsigned row) const {
    if (group == 0) return row * stride;
    const unsigned g = row / group;
    return g * group_stride + (row - g * group) * stride;
  }
};

// Where a row's 16-byte vectors begin and how many there are; `head` elements stand in front of them, `tail` behind.
template <typename T>
struct Cut {
  int head, vectors, tail;
  __device__ __forceinline__ Cut(const T* x, int vocab) {
    constexpr int E = Vec<T>::kElements;
    head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
    if (head > vocab) head = vocab;
    vectors = (vocab - head) / E;
    tail = vocab - head - vectors * E;
  }
  // Element outside the vectors that thread `i` looks after (the first 8 threads in front, the next 8 behind), or -1.
  __device__ __forceinline__ int loose(int i, int vocab) const {
    return i < 8 ? (i < head ? i : -1) : (i < 16 && i - 8 < tail ? vocab - tail + i - 8 : -1);
  }
};

// Zeros for elements [begin, end), by `count` threads of which this is thread `i`.
template <typename T>
__device__ __forceinline__ void clear(T* g, int begin, int end, int i, int count) {
  const Cut<T> cut(g + begin, end - begin);
  const int own = i < 16 ? cut.loose(i, end - begin) : -1;
  if (own >= 0) store1(g + begin + own, 0.f);
  uint4* p = reinterpret_cast<uint4*>(g + begin + cut.head);
  for (int v = i; v < cut.vectors; v += count) __stcs(p + v, make_uint4(0, 0, 0, 0));
}

// A vector of gradients to elements that begin at `g`: one store where the gradient is cut like the logits.
template <typename T>
__device__ __forceinline__ void put(T* g, const uint4& q, bool same_cut) {
  if (same_cut) {
    __stcs(reinterpret_cast<uint4*>(g), q);
  } else {
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < Vec<T>::kElements; ++i) g[i] = e[i];
  }
}

template <typename T>
__device__ __forceinline__ bool cut_alike(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

// Log-probabilities alone: a row per block, or per cluster of blocks when there are too few rows to fill the device.  HBM-bound:
// 2048 rows of 151936 bf16 logits take 96 us (6.5 TB/s), 8192 of them 0.41 ms; exp2 keeps the special-function units 73 % busy
// meanwhile.  One pass with a running reference and sum, 4 vectors per thread in flight and full occupancy; for rows this
// long 256 threads were 2-4 % slower than 512, and 8 vectors in flight 10 %.
template <typename T, int THREADS, int NB, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    row_kernel(const T* __restrict__ logits, Layout layout, const long long* __restrict__ ids, float inv_t,
               float* __restrict__ logprob, float2* __restrict__ stats, int vocab) {
  const unsigned size = cluster_size(), rank = cluster_rank();
  const long long row = blockIdx.x / size, t = ids[row];
  const T* x = logits + layout.of((unsigned)row);
  const int first = rank * THREADS + threadIdx.x, step = size * THREADS;
  if (t < 0 || t >= vocab) {
    if (first == 0) {
      logprob[row] = 0.f;
      if (stats != nullptr) stats[row] = make_float2(0.f, 0.f);
    }
    return;
  }
  if (size > 1) cluster_arrive();
  const Cut<T> cut(x, vocab);
  const uint4* p = reinterpret_cast<const uint4*>(x + cut.head);
  const int loose = first < 16 ? cut.loose(first, vocab) : -1;
  const float xt = load1(x + t);
  Running run;
  run.c = inv_t * kLog2e;
  int v = first;
  for (; v + (NB - 1) * step < cut.vectors; v += NB * step) {
    uint4 q[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) q[j] = __ldcs(p + v + j * step);
    run.template take<T, NB>(q);
  }
  for (; v < cut.vectors; v += step) {
    const uint4 q[1] = {__ldcs(p + v)};
    run.template take<T, 1>(q);
  }
  if (loose >= 0) run.take_one(load1(x + loose));
  const float2 sums = halves(run.s);
  float m = run.m, s = sums.x + sums.y;
  row_join<THREADS>(m, s, run.c, rank, size);
  if (first == 0) {
    const float log2_s = log2f(s);
    logprob[row] = (xt - m) * inv_t - log2_s * kLn2;
    if (stats != nullptr) stats[row] = make_float2(m, log2_s);
  }
}

__device__ __forceinline__ void copy_async(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Log-probabilities and gradient in one kernel.  Bound by HBM in principle (each logit read and each gradient written
// once) and by latency in practice, since no gradient can be formed before the whole row has been seen.  A row does not fit
// one SM (151936 bf16 logits are 304 KB), so a cluster of blocks shares it, and the second pass reads it again from the L2:
// 5 blocks of 256 threads per SM, at most 20 vectors per thread, keep 60 MB of rows in flight.  What keeps the loads going is
// a ring of kRing batches of kRingBatch vectors per thread in shared memory, filled by asynchronous copies that each thread
// makes for itself (no barrier): the first pass runs it upwards, the second one downwards, beginning with the batches that
// it still holds.  The ring is unrolled and the cluster's size a constant, so that a batch of 16 elements costs few
// instructions beside its arithmetic (27 per pair of elements in all; 38 with computed slots and addresses, which took
// 225 us and drew more power).  2048 rows of 151936 bf16: 212 us, 205 in place, where a copy of the same bytes takes 195;
// 8192 rows 0.81 ms in a short run of calls, 0.84-0.95 in long ones, by how far the power cap lowers the clock.  Other forms, same 2048 rows: loads
// through registers 232 us, rows held in the registers of a cluster 291-388, in its shared memory 253-390 (the join of the
// row then leaves the memory idle), persistent blocks that fetch their next row early 231-296, two kernels (forward, then
// backward_kernel) 280.
constexpr int kRing = 5, kRingBatch = 2;

template <typename T, int THREADS, int CLUSTER, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    row_grad_kernel(const T* logits, Layout layout, const long long* __restrict__ ids, const float* __restrict__ weight,
                    float inv_t, float* __restrict__ logprob, T* grad, long long grad_stride, int vocab) {
  constexpr int E = Vec<T>::kElements, B = kRingBatch, R = kRing, kStep = CLUSTER * THREADS, kBatch = B * kStep;
  extern __shared__ uint4 ring[];   // [R * B][THREADS]
  const unsigned rank = CLUSTER > 1 ? cluster_rank() : 0;
  const long long row = blockIdx.x / CLUSTER, t = ids[row];
  const T* x = logits + layout.of((unsigned)row);
  T* g = grad + row * grad_stride;
  const int first = rank * THREADS + threadIdx.x;
  if (t < 0 || t >= vocab) {
    if (first == 0) logprob[row] = 0.f;
    clear(g, 0, vocab, first, kStep);
    return;
  }
  if (CLUSTER > 1) cluster_arrive();
  const Cut<T> cut(x, vocab);
  // batches of B vectors per thread: `whole` that every thread has in full, and one more where some vectors are missing
  const int whole = cut.vectors / kBatch, left = cut.vectors - whole * kBatch;
  const uint4* from = reinterpret_cast<const uint4*>(x + cut.head) + first;   // the next batch to be fetched
  uint4* const mine = ring + threadIdx.x;
  const auto fetch = [&](int r) {
#pragma unroll
    for (int j = 0; j < B; ++j) copy_async(mine + (r * B + j) * THREADS, from + j * kStep);
  };
  const auto fetch_partial = [&](int r) {
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (first + j * kStep < left) copy_async(mine + (r * B + j) * THREADS, from + j * kStep);
  };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r < whole) fetch(r);
    else if (r == whole) fetch_partial(r);
    copy_commit();
    from += kBatch;
  }
  const int loose = first < 16 ? cut.loose(first, vocab) : -1;
  const float loose_x = loose >= 0 ? load1(x + loose) : 0.f;
  const float xt = load1(x + t);   // by all: before any of it may be overwritten
  const float w = (weight != nullptr ? weight[row] : 1.f) * inv_t;
  Running run;
  run.c = inv_t * kLog2e;
  const auto take = [&](int r) {
    copy_wait<R - 1>();
    uint4 q[B];
#pragma unroll
    for (int j = 0; j < B; ++j) q[j] = mine[(r * B + j) * THREADS];
    run.template take_lazily<T, B>(q);
  };
  int k = 0;
  for (; k + R <= whole; k += R) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      take(r);
      if (k + r + R < whole) fetch(r);   // into the slot that has just been read
      else if (k + r + R == whole) fetch_partial(r);
      copy_commit();
      from += kBatch;
    }
  }
  const int rest = whole - k;   // batches behind the last full round of the ring; the partial one is number `rest` of this round
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r < rest) {
      take(r);
      copy_commit();
    } else if (r == rest && left > 0) {
      copy_wait<0>();
#pragma unroll
      for (int j = 0; j < B; ++j)
        if (first + j * kStep < left) {
          const uint4 q[1] = {mine[(r * B + j) * THREADS]};
          run.template take_lazily<T, 1>(q);
        }
    }
  }
  if (loose >= 0) run.take_one(loose_x);
  const float2 sums = halves(run.s);
  float m = run.m, s = sums.x + sums.y;
  row_join<THREADS>(m, s, run.c, rank, CLUSTER);
  const float log2_s = log2f(s);
  const float l = (xt - m) * inv_t - log2_s * kLn2;
  if (first == 0) logprob[row] = l;
  const pair_t cc = pair(run.c, run.c), less = pair(-log2_s, -log2_s), scale = pair(-w, -w);
  const auto f = [&](pair_t d) { return mul2(exp2_2(fma2(d, cc, less)), scale); };
  const bool alike = cut_alike(x, g);
  const long long behind = (long long)whole * kBatch;
  T* to = g + cut.head + (behind + first) * E;                                                      // the batch given next
  from = reinterpret_cast<const uint4*>(x + cut.head) + first + (behind - (long long)R * kBatch);   // R batches before it
  const auto give = [&](int r, int j) { put(to + j * (kStep * E), Vec<T>::map(mine[(r * B + j) * THREADS], m, f), alike); };
  const auto give_batch = [&](int r) {
    to -= kBatch * E;
    from -= kBatch;
    copy_wait<R - 1>();
#pragma unroll
    for (int j = 0; j < B; ++j) give(r, j);
    if (k > 0) fetch(r);
    copy_commit();
  };
  copy_wait<0>();
#pragma unroll
  for (int r = R - 1; r >= 0; --r) {
    if (r < rest) {
      give_batch(r);
    } else if (r == rest && left > 0) {
#pragma unroll
      for (int j = 0; j < B; ++j)
        if (first + j * kStep < left) give(r, j);
      if (k > 0) fetch(r);
      copy_commit();
    }
  }
  for (k -= R; k >= 0; k -= R) {
#pragma unroll
    for (int r = R - 1; r >= 0; --r) give_batch(r);
  }
  if (loose >= 0) store1(g + loose, exp2_fast((loose_x - m) * run.c - log2_s) * -w);
  // the target's own column, by the thread that has just written it: 1 - p without the cancellation
  const int at = (int)t - cut.head;
  const bool own = at >= 0 && at / E < cut.vectors ? at / E % kStep == first : loose == (int)t;
  if (own) store1(g + t, -expm1f(l) * w);
}

// The backward pass on its own: p from the forward's two numbers per row, one read and one write per logit, nothing shared
// between threads.  HBM-bound: 4096 x 50304 bf16 takes 124 us (6.66 TB/s), 8192 x 32000 fp32 305 us (6.9 TB/s, some of it from
// the L2).  A block takes 4 vectors per thread of one row: no loop, many blocks, reads and writes spread evenly (a copy
// written like this reaches 6.7 TB/s, one with a fixed grid that loops 6.0).  Rows of ignored ids are only cleared.
constexpr int kBackVectors = 4;

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) backward_kernel(const T* logits, Layout layout,
                                                           const long long* __restrict__ ids, const float2* __restrict__ stats,
                                                           const float* __restrict__ grad_logprob, float inv_t, T* grad,
                                                           long long grad_stride, int vocab, int parts) {
  constexpr int E = Vec<T>::kElements, kPart = THREADS * kBackVectors;
  const long long row = blockIdx.x / parts, t = ids[row];
  const int part = blockIdx.x - row * parts;
  const T* x = logits + layout.of((unsigned)row);
  T* g = grad + row * grad_stride;
  const Cut<T> cut(x, vocab);
  const bool last = part == parts - 1;
  if (t < 0 || t >= vocab) {
    clear(g, part == 0 ? 0 : min(vocab, cut.head + part * kPart * E), last ? vocab : min(vocab, cut.head + (part + 1) * kPart * E),
          threadIdx.x, THREADS);
    return;
  }
  const uint4* p = reinterpret_cast<const uint4*>(x + cut.head);
  const int first = part * kPart + threadIdx.x, end = min(cut.vectors, (part + 1) * kPart);
  uint4 q[kBackVectors];
#pragma unroll
  for (int j = 0; j < kBackVectors; ++j)
    if (first + j * THREADS < end) q[j] = __ldcs(p + first + j * THREADS);
  const float c = inv_t * kLog2e, w = grad_logprob[row] * inv_t;
  const float2 st = stats[row];
  const pair_t cc = pair(c, c), less = pair(-st.y, -st.y), scale = pair(-w, -w);
  const auto f = [&](pair_t d) { return mul2(exp2_2(fma2(d, cc, less)), scale); };
  const bool alike = cut_alike(x, g);
  const int at = (int)t - cut.head, holder = at / E;
  const bool inside = at >= 0 && holder < cut.vectors;
#pragma unroll
  for (int j = 0; j < kBackVectors; ++j) {
    const int v = first + j * THREADS;
    if (v < end) {
      const bool own = inside && v == holder;
      const float xt = own ? load1(x + t) : 0.f;   // before it may be overwritten
      put(g + cut.head + (long long)v * E, Vec<T>::map(q[j], st.x, f), alike);
      if (own) store1(g + t, -expm1f((xt - st.x) * inv_t - st.y * kLn2) * w);
    }
  }
  // the elements in front of the vectors belong to the first part, those behind to the last
  const int loose = threadIdx.x < 16 ? cut.loose(threadIdx.x, vocab) : -1;
  if (loose >= 0 && (threadIdx.x < 8 ? part == 0 : last)) {
    const float xv = load1(x + loose);
    store1(g + loose, loose == (int)t ? -expm1f((xv - st.x) * inv_t - st.y * kLn2) * w
                                      : exp2_fast((xv - st.x) * c - st.y) * -w);
  }
}

int check_rows(const char* who, const void* logits, int dtype, int64_t row_stride, int64_t group_rows, int64_t group_stride,
               const int64_t* ids, float temperature, int64_t rows, int64_t vocab) {
  MOLT_REQUIRE(rows >= 0 && vocab > 0, MOLT_E_VALUE, "%s: bad shape", who);
  MOLT_REQUIRE(rows <= (1LL << 27) && vocab <= (1LL << 30), MOLT_E_CAPABILITY, "%s: more than 2^27 rows or 2^30 columns", who);
  MOLT_REQUIRE(dtype == MOLT_DTYPE_BF16 || dtype == MOLT_DTYPE_F32, MOLT_E_CAPABILITY, "%s: logits must be bf16 or fp32", who);
  // well inside fp32, with log2(e) / T and the slack of the running reference
  MOLT_REQUIRE(temperature >= 1e-30f && temperature <= 1e30f, MOLT_E_VALUE, "%s: temperature must lie in [1e-30, 1e30]", who);
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logits && ids, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(ids) % 8 == 0, MOLT_E_VALUE, "%s: token_ids are not aligned to their type", who);
  MOLT_REQUIRE(row_stride == 0 || row_stride >= vocab, MOLT_E_VALUE, "%s: rows of logits overlap", who);
  MOLT_REQUIRE(group_rows >= 0, MOLT_E_VALUE, "%s: bad group_rows", who);
  MOLT_REQUIRE(group_rows == 0 || group_stride == 0 || group_stride >= vocab, MOLT_E_VALUE, "%s: groups of logits overlap", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == MOLT_DTYPE_BF16 ? 2 : 4) == 0, MOLT_E_VALUE,
               "%s: logits are not aligned to their type", who);
  return MOLT_OK;
}

// The gradient may lie over the logits exactly, or beside them (also in other columns of the same wider rows).
int check_grad(const char* who, const void* logits, int dtype, const Layout& layout, const void* grad, int64_t grad_stride, int64_t rows,
               int64_t vocab) {
  if (rows == 0) return MOLT_OK;
  const int64_t size = dtype == MOLT_DTYPE_BF16 ? 2 : 4;
  MOLT_REQUIRE(grad != nullptr, MOLT_E_VALUE, "%s: NULL gradient pointer", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(grad) % size == 0, MOLT_E_VALUE, "%s: the gradient is not aligned to its type", who);
  MOLT_REQUIRE(grad_stride >= vocab, MOLT_E_VALUE, "%s: rows of the gradient overlap", who);
  const intptr_t a = reinterpret_cast<intptr_t>(logits), b = reinterpret_cast<intptr_t>(grad);
  const bool alike = layout.group == 0 && layout.stride == grad_stride;
  if (a == b && (alike || rows == 1)) return MOLT_OK;
  const int64_t groups = layout.group == 0 ? 1 : (rows - 1) / layout.group + 1, in_group = layout.group == 0 ? rows : layout.group;
  const intptr_t a_end = a + ((groups - 1) * layout.group_stride + (in_group - 1) * layout.stride + vocab) * size;
  const intptr_t b_end = b + ((rows - 1) * grad_stride + vocab) * size;
  if (a_end <= b || b_end <= a) return MOLT_OK;
  if (alike) {
    const intptr_t pitch = grad_stride * size, shift = (((b - a) % pitch) + pitch) % pitch;
    if (shift >= vocab * size && shift <= pitch - vocab * size) return MOLT_OK;
  }
  return fail(MOLT_E_VALUE, "%s: the gradient overlaps the logits without being the same rows", who);
}

// Rows of one group, or of groups that follow each other like their rows, need no division.
Layout layout_of(int64_t row_stride, int64_t group_rows, int64_t group_stride, int64_t rows) {
  const bool one = group_rows == 0 || group_rows >= rows || group_stride == group_rows * row_stride;
  return {row_stride, one ? 0 : group_stride, one ? 0u : (unsigned)group_rows};
}

template <typename... Params, typename... Args>
int launch_clusters(const char* what, void (*kernel)(Params...), int64_t rows, int cluster, int threads, size_t shared, cudaStream_t s,
                    Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(rows * cluster));
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&config, kernel, Params(args)...);
  return launch_status(what);
}

// Threads for a row of `vectors` 16-byte vectors.  A block that is done too soon spends its time on being launched, on its
// first loads and on its join: it is made as small as leaves a thread 13 vectors (16384 rows x 8192 bf16, forward: 99 us with
// 512 threads, 46 with 64), but not so small that there are too few threads for the device (while a thread keeps 4).
int threads_for(int64_t rows, int64_t vectors, int most, int resident) {
  int threads = 64;
  while (threads < most && vectors >= 2 * threads * 13) threads *= 2;
  while (threads < most && rows * threads < (int64_t)148 * resident && vectors >= 2 * threads * 4) threads *= 2;
  return threads;
}

// Where the largest block would not do, a cluster of them takes a row (a power of two, at most 8):
// * with gradient, until a thread has at most 20 vectors, so that the rows in flight stay in the L2;
// * in both directions, as long as the rows alone do not fill the device and a thread keeps at least 4 vectors.
template <typename T>
int launch_forward(const void* logits, const Layout& layout, const int64_t* ids, float temperature, float* logprob, float* stats,
                   int64_t rows, int64_t vocab, cudaStream_t s) {
  constexpr int kResident = sizeof(T) == 2 ? 2048 : 1536;   // threads per SM: 32 registers each, or 40
  const int64_t vectors = vocab / Vec<T>::kElements;
  const int threads = threads_for(rows, vectors, 512, kResident);
  const auto launch = [&](auto kernel, int cluster) {
    return launch_clusters("token_logprob row_kernel", kernel, rows, cluster, threads, 0, s, reinterpret_cast<const T*>(logits), layout,
                           reinterpret_cast<const long long*>(ids), 1.f / temperature, logprob, reinterpret_cast<float2*>(stats), vocab);
  };
  if (threads == 64) return launch(row_kernel<T, 64, 4, kResident / 64>, 1);
  if (threads == 128) return launch(row_kernel<T, 128, 4, kResident / 128>, 1);
  if (threads == 256) return launch(row_kernel<T, 256, 4, kResident / 256>, 1);
  int cluster = 1;
  while (cluster < 8 && rows * cluster < 148 * 2 && vectors >= cluster * 512 * 4) cluster *= 2;
  return launch(row_kernel<T, 512, 4, kResident / 512>, cluster);
}

template <typename T>
int launch_grad(const void* logits, const Layout& layout, const int64_t* ids, const float* weight, float temperature, float* logprob,
                void* grad, int64_t grad_stride, int64_t rows, int64_t vocab, cudaStream_t s) {
  constexpr int kResident = 1280;   // threads per SM: 48 registers and 160 bytes of the ring each
  const int64_t vectors = vocab / Vec<T>::kElements;
  const int threads = threads_for(rows, vectors, 256, kResident);
  const auto launch = [&](auto kernel, int cluster) {
    return launch_clusters("token_logprob row_grad_kernel", kernel, rows, cluster, threads, threads * kRing * kRingBatch * sizeof(uint4), s,
                           reinterpret_cast<const T*>(logits), layout, reinterpret_cast<const long long*>(ids), weight,
                           1.f / temperature, logprob, reinterpret_cast<T*>(grad), grad_stride, vocab);
  };
  if (threads == 64) return launch(row_grad_kernel<T, 64, 1, kResident / 64>, 1);
  if (threads == 128) return launch(row_grad_kernel<T, 128, 1, kResident / 128>, 1);
  int cluster = 1;
  while (cluster < 8 && (vectors > cluster * 256 * 20 || (rows * cluster < 148 * 4 && vectors >= cluster * 256 * 4))) cluster *= 2;
  if (cluster == 1) return launch(row_grad_kernel<T, 256, 1, kResident / 256>, 1);
  if (cluster == 2) return launch(row_grad_kernel<T, 256, 2, kResident / 256>, 2);
  if (cluster == 4) return launch(row_grad_kernel<T, 256, 4, kResident / 256>, 4);
  return launch(row_grad_kernel<T, 256, 8, kResident / 256>, 8);
}

// Small blocks where a row would leave most of a large one idle (16384 x 500 bf16: 29 us with 256 threads, 13 with 64).
template <typename T>
int launch_backward(const char* who, const void* logits, const Layout& layout, const int64_t* ids, const float* stats,
                    const float* grad_logprob, float temperature, void* grad, int64_t grad_stride, int64_t rows, int64_t vocab,
                    cudaStream_t s) {
  const int threads = vocab / Vec<T>::kElements <= 64 * kBackVectors ? 64 : 256;
  const int64_t part = (int64_t)threads * kBackVectors * Vec<T>::kElements, parts = (vocab + part - 1) / part;
  MOLT_REQUIRE(rows * parts < (1LL << 31), MOLT_E_CAPABILITY, "%s: more than 2^31 blocks of logits", who);
  const auto kernel = threads == 64 ? backward_kernel<T, 64> : backward_kernel<T, 256>;
  kernel<<<(unsigned)(rows * parts), threads, 0, s>>>(
      reinterpret_cast<const T*>(logits), layout, reinterpret_cast<const long long*>(ids), reinterpret_cast<const float2*>(stats),
      grad_logprob, 1.f / temperature, reinterpret_cast<T*>(grad), grad_stride, (int)vocab, (int)parts);
  return launch_status("token_logprob backward_kernel");
}

}  // namespace
}  // namespace molt

using namespace molt;

extern "C" int molt_token_logprob_fwd(const void* logits, int dtype, int64_t row_stride, int64_t group_rows,
                                      int64_t group_stride, const int64_t* token_ids, float temperature, float* logprob,
                                      float* stats, int64_t rows, int64_t vocab, uintptr_t stream) {
  const char* who = "molt_token_logprob_fwd";
  if (int rc = check_rows(who, logits, dtype, row_stride, group_rows, group_stride, token_ids, temperature, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logprob != nullptr, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, MOLT_E_VALUE, "%s: stats must be 8-byte aligned", who);
  const Layout layout = layout_of(row_stride, group_rows, group_stride, rows);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MOLT_DTYPE_BF16
             ? launch_forward<__nv_bfloat16>(logits, layout, token_ids, temperature, logprob, stats, rows, vocab, s)
             : launch_forward<float>(logits, layout, token_ids, temperature, logprob, stats, rows, vocab, s);
}

extern "C" int molt_token_logprob_grad(const void* logits, int dtype, int64_t row_stride, int64_t group_rows,
                                       int64_t group_stride, const int64_t* token_ids, const float* weight, float temperature,
                                       float* logprob, void* grad_logits, int64_t grad_stride, int64_t rows, int64_t vocab,
                                       uintptr_t stream) {
  const char* who = "molt_token_logprob_grad";
  if (int rc = check_rows(who, logits, dtype, row_stride, group_rows, group_stride, token_ids, temperature, rows, vocab)) return rc;
  const Layout layout = layout_of(row_stride, group_rows, group_stride, rows);
  if (int rc = check_grad(who, logits, dtype, layout, grad_logits, grad_stride, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logprob != nullptr, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MOLT_DTYPE_BF16 ? launch_grad<__nv_bfloat16>(logits, layout, token_ids, weight, temperature, logprob, grad_logits,
                                                               grad_stride, rows, vocab, s)
                                  : launch_grad<float>(logits, layout, token_ids, weight, temperature, logprob, grad_logits,
                                                       grad_stride, rows, vocab, s);
}

extern "C" int molt_token_logprob_bwd(const void* logits, int dtype, int64_t row_stride, int64_t group_rows,
                                      int64_t group_stride, const int64_t* token_ids, const float* stats,
                                      const float* grad_logprob, float temperature, void* grad_logits, int64_t grad_stride,
                                      int64_t rows, int64_t vocab, uintptr_t stream) {
  const char* who = "molt_token_logprob_bwd";
  if (int rc = check_rows(who, logits, dtype, row_stride, group_rows, group_stride, token_ids, temperature, rows, vocab)) return rc;
  const Layout layout = layout_of(row_stride, group_rows, group_stride, rows);
  if (int rc = check_grad(who, logits, dtype, layout, grad_logits, grad_stride, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(stats && grad_logprob, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, MOLT_E_VALUE, "%s: stats must be 8-byte aligned", who);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MOLT_DTYPE_BF16 ? launch_backward<__nv_bfloat16>(who, logits, layout, token_ids, stats, grad_logprob, temperature,
                                                                   grad_logits, grad_stride, rows, vocab, s)
                                  : launch_backward<float>(who, logits, layout, token_ids, stats, grad_logprob, temperature,
                                                           grad_logits, grad_stride, rows, vocab, s);
}

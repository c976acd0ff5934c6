// Global norm of a list of gradients, the clipping coefficient, and the clipped gradients.
//   norm = (sum g^2)^(1/2)  or  max |g|;   coefficient = min(1, max_norm / (norm + 1e-6));   out = g * coefficient
// The list travels in the kernel's parameters (no copy to the device, nothing kept, capture-safe); a list longer than a
// table is walked in several launches.  Every tensor is cut into chunks, the chunks of the list are numbered through, and
// block i of G takes chunks i, i + G, ...; it leaves one partial sum, and the partial sums are added in a fixed order, so a
// list gives the same bits on every call.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.cuh"

namespace molt {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;         // elements of a chunk
constexpr int kBlocks = 148 * 5;     // most partial sums of one table; a fixed figure, it decides which chunks one of them holds
constexpr int kScaleBlocks = 148 * 32;   // many more than run at a time: blocks that begin late even out the others
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread

template <int CAPACITY>
struct Table {
  const void* grad[CAPACITY];
  void* out[CAPACITY];
  long long elements[CAPACITY];
  unsigned first[CAPACITY + 1];      // number of a tensor's first chunk; [count] = all chunks
  unsigned char half[CAPACITY];      // bf16
  int count;
};
constexpr int kTable = 1024;         // tensors per launch: the table must stay below the 32764 bytes of kernel parameters
constexpr int kSmallTable = 16;      // a short list, such as one arena, does not carry 30 KB to the device
static_assert(sizeof(Table<kTable>) < 32000, "kernel parameters");

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ double larger(double a, double b) { return isnan(a) || isnan(b) ? (double)NAN : fmax(a, b); }

template <bool MAX>
__device__ __forceinline__ double block_total(double v) {
  __shared__ double part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double other = __shfl_xor_sync(~0u, v, o);
    v = MAX ? larger(v, other) : v + other;
  }
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < warps; ++w) v = MAX ? larger(v, part[w]) : v + part[w];
  return v;
}

// The tensor that chunk `c` belongs to.
template <int CAPACITY>
__device__ __forceinline__ int tensor_of(const Table<CAPACITY>& table, unsigned c) {
  int low = 0, high = table.count - 1;
  while (low < high) {
    const int middle = (low + high + 1) >> 1;
    if (table.first[middle] <= c) low = middle;
    else high = middle - 1;
  }
  return low;
}

// The elements of 16 bytes.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kElements = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kElements = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};

// A stretch of elements: those in front of its 16-byte vectors, the vectors, those behind.
template <typename T>
struct Cut {
  int head, vectors, tail;
  __device__ __forceinline__ Cut(const T* g, int n) {
    head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / sizeof(T)));
    vectors = (n - head) / Vec<T>::kElements;
    tail = n - head - vectors * Vec<T>::kElements;
  }
  // The element outside the vectors that this thread looks after, or -1.
  __device__ __forceinline__ int loose(int n) const {
    const int i = threadIdx.x;
    return i < 8 ? (i < head ? i : -1) : (i < 16 && i - 8 < tail ? n - tail + i - 8 : -1);
  }
};

// Squares of one vector: in fp32 where neither a square nor their sum leaves its range (the sum of at most 8 is then
// within 10 roundings), else in 64 bits.  Below 2^-80 a square may have been flushed that is not small beside the others.
template <int N>
__device__ __forceinline__ double squares(const float (&v)[N], const uint4& q) {
  float a = v[0] * v[0], b = v[1] * v[1];
#pragma unroll
  for (int i = 2; i < N; i += 2) {
    a = fmaf(v[i], v[i], a);
    b = fmaf(v[i + 1], v[i + 1], b);
  }
  const float sum = a + b;
  if (sum >= 0x1p-80f && sum <= 0x1.fffffep127f) return sum;
  if ((q.x | q.y | q.z | q.w) == 0u) return 0.;
  double exact = 0.;
#pragma unroll
  for (int i = 0; i < N; ++i) exact += (double)v[i] * (double)v[i];
  return exact;
}

template <int N>
__device__ __forceinline__ float magnitude(const float (&v)[N]) {   // NaN if there is one
  float top = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[i])));
  return top;
}

template <bool MAX, typename T>
__device__ __forceinline__ double chunk_total(const T* g, int n, double acc) {
  constexpr int E = Vec<T>::kElements;
  const Cut<T> cut(g, n);
  const uint4* p = reinterpret_cast<const uint4*>(g + cut.head);
  for (int v = threadIdx.x; v < cut.vectors; v += kUnroll * kThreads) {
    uint4 q[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) q[j] = v + j * kThreads < cut.vectors ? p[v + j * kThreads] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float x[E];
      Vec<T>::unpack(q[j], x);
      if (MAX) acc = larger(acc, (double)magnitude(x));
      else acc += squares(x, q[j]);
    }
  }
  const int own = cut.loose(n);
  if (own >= 0) {
    const double x = load1(g + own);
    acc = MAX ? larger(acc, fabs(x)) : acc + x * x;
  }
  return acc;
}

// HBM-bound: 742 MB in 84 tensors take 112 us (6.6 TB/s), a 74 MB arena 14.7 us (8.5 where the L2 holds it already).  8 loads in flight per thread, 4096 or 16384
// elements per chunk and more blocks were each within 5 %, or slower.
template <bool MAX, int CAPACITY>
__global__ void __launch_bounds__(kThreads, 5) norm_kernel(const __grid_constant__ Table<CAPACITY> table,
                                                        double* __restrict__ part) {
  let_next_begin();   // it waits for the partial sums itself
  double acc = 0.;
  const unsigned chunks = table.first[table.count];
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int k = tensor_of(table, c);
    const long long begin = (long long)(c - table.first[k]) * kChunk;
    const int n = (int)min((long long)kChunk, table.elements[k] - begin);
    acc = table.half[k] ? chunk_total<MAX>(reinterpret_cast<const __nv_bfloat16*>(table.grad[k]) + begin, n, acc)
                        : chunk_total<MAX>(reinterpret_cast<const float*>(table.grad[k]) + begin, n, acc);
  }
  acc = block_total<MAX>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The norm and the coefficient from the partial sums, by one block; every thread gets them.
template <bool MAX>
__device__ __forceinline__ float2 finish(const Written part, int parts, float grad_scale, float max_norm) {
  double acc = 0.;
  for (int i = threadIdx.x; i < parts; i += kUnroll * blockDim.x) {
    double v[kUnroll];   // all requested before the first is used: volatile loads are not moved together
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) v[j] = i + j * blockDim.x < parts ? part[i + j * blockDim.x] : 0.;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) acc = MAX ? larger(acc, v[j]) : acc + v[j];
  }
  acc = block_total<MAX>(acc);
  // The norm of finite gradients may be beyond fp32: the coefficient comes from the 64-bit norm, and the norm is reported as
  // fp32's largest value, so that only a gradient that is not finite gives a norm that is not.
  const double norm = (MAX ? acc : sqrt(acc)) * fabs((double)grad_scale);
  const double c = (double)max_norm / (norm + 1e-6);
  const float reported = norm > (double)FLT_MAX && !isinf(norm) ? FLT_MAX : (float)norm;
  return make_float2(reported, c > 1. ? 1.f : (float)c);   // NaN stays
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const Written part, int parts, float grad_scale,
                                                               float max_norm, float* __restrict__ result) {
  wait_for_previous();
  const float2 r = finish<MAX>(part, parts, grad_scale, max_norm);
  if (threadIdx.x == 0) {
    result[0] = r.x;
    result[1] = r.y;
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* g, T* out, int n, float c) {
  constexpr int E = Vec<T>::kElements;
  const Cut<T> cut(g, n);
  const uint4* p = reinterpret_cast<const uint4*>(g + cut.head);
  if (((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
    uint4* to = reinterpret_cast<uint4*>(out + cut.head);
    for (int v = threadIdx.x; v < cut.vectors; v += kUnroll * kThreads) {
      uint4 q[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (v + j * kThreads < cut.vectors) q[j] = __ldcs(p + v + j * kThreads);
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        float x[E];
        Vec<T>::unpack(q[j], x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] *= c;
        if (v + j * kThreads < cut.vectors) __stcs(to + v + j * kThreads, Vec<T>::pack(x));
      }
    }
  } else {   // an output cut elsewhere than its gradient: element by element
    for (int i = cut.head + threadIdx.x; i < n - cut.tail; i += kThreads) store1(out + i, load1(g + i) * c);
  }
  const int own = cut.loose(n);
  if (own >= 0) store1(out + own, load1(g + own) * c);
}

// Every block adds the partial sums up for itself (they lie in the L2) instead of waiting for one that does.  The chunks
// are taken from the last to the first: what the norm read last is what the L2 still holds.  HBM-bound: 742 MB read and
// written take 220 us (6.7 TB/s), the 74 MB arena 22 us.
template <bool MAX, int CAPACITY>
__global__ void __launch_bounds__(kThreads, 4) scale_kernel(const __grid_constant__ Table<CAPACITY> table,
                                                         const Written part, int parts, float max_norm,
                                                         float* __restrict__ result) {
  wait_for_previous();
  const float2 r = finish<MAX>(part, parts, 1.f, max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    result[0] = r.x;
    result[1] = r.y;
  }
  const unsigned chunks = table.first[table.count];
  for (unsigned i = blockIdx.x; i < chunks; i += gridDim.x) {
    const unsigned c = chunks - 1 - i;
    const int k = tensor_of(table, c);
    const long long begin = (long long)(c - table.first[k]) * kChunk;
    const int n = (int)min((long long)kChunk, table.elements[k] - begin);
    if (table.half[k])
      chunk_scale(reinterpret_cast<const __nv_bfloat16*>(table.grad[k]) + begin,
                  reinterpret_cast<__nv_bfloat16*>(table.out[k]) + begin, n, r.y);
    else
      chunk_scale(reinterpret_cast<const float*>(table.grad[k]) + begin, reinterpret_cast<float*>(table.out[k]) + begin, n, r.y);
  }
}

int tables_of(int count) { return (count + kTable - 1) / kTable; }

// Fills `table` with items [begin, begin + n).
template <int CAPACITY>
void fill(Table<CAPACITY>& table, const molt_grad_item* items, int n) {
  table.count = n;
  unsigned chunks = 0;
  for (int k = 0; k < n; ++k) {
    table.grad[k] = items[k].grad;
    table.out[k] = items[k].out;
    table.elements[k] = items[k].count;
    table.half[k] = items[k].dtype == MOLT_DTYPE_BF16;
    table.first[k] = chunks;
    chunks += (unsigned)((items[k].count + kChunk - 1) / kChunk);
  }
  table.first[n] = chunks;
}

template <bool MAX>
int launch_norm(const molt_grad_item* items, int n, int blocks, double* part, cudaStream_t s) {
  if (n <= kSmallTable) {
    Table<kSmallTable> table;
    fill(table, items, n);
    norm_kernel<MAX><<<blocks, kThreads, 0, s>>>(table, part);
  } else {
    Table<kTable> table;
    fill(table, items, n);
    norm_kernel<MAX><<<blocks, kThreads, 0, s>>>(table, part);
  }
  return launch_status("norm_kernel");
}

template <bool MAX>
int launch_scale(const molt_grad_item* items, int n, int blocks, const double* part, int parts, float max_norm, float* result,
                 cudaStream_t s) {
  if (n <= kSmallTable) {
    Table<kSmallTable> table;
    fill(table, items, n);
    launch_behind(scale_kernel<MAX, kSmallTable>, blocks, kThreads, s, table, part, parts, max_norm, result);
  } else {
    Table<kTable> table;
    fill(table, items, n);
    launch_behind(scale_kernel<MAX, kTable>, blocks, kThreads, s, table, part, parts, max_norm, result);
  }
  return launch_status("scale_kernel");
}

// Blocks for the chunks of a table, at least one.
int blocks_for(const molt_grad_item* items, int n, int most) {
  long long chunks = 0;
  for (int k = 0; k < n; ++k) chunks += (items[k].count + kChunk - 1) / kChunk;
  return (int)std::max(1LL, std::min((long long)most, chunks));
}

struct Span {
  uintptr_t begin, end;
  int item;
  bool written;
};

int check_items(const char* who, const molt_grad_item* items, int count, bool clip) {
  MOLT_REQUIRE(count > 0 && items != nullptr, MOLT_E_VALUE, "%s: no gradient", who);
  long long chunks = 0;
  for (int k = 0; k < count; ++k) {
    const molt_grad_item& it = items[k];
    MOLT_REQUIRE(it.dtype == MOLT_DTYPE_BF16 || it.dtype == MOLT_DTYPE_F32, MOLT_E_CAPABILITY,
                 "%s: gradients must be bf16 or fp32", who);
    const uintptr_t size = it.dtype == MOLT_DTYPE_BF16 ? 2 : 4;
    MOLT_REQUIRE(it.count >= 0 && it.count <= (1LL << 42), MOLT_E_VALUE, "%s: bad element count of gradient %d", who, k);
    MOLT_REQUIRE(it.count == 0 || (it.grad != nullptr && (!clip || it.out != nullptr)), MOLT_E_VALUE, "%s: gradient %d is NULL",
                 who, k);
    MOLT_REQUIRE(reinterpret_cast<uintptr_t>(it.grad) % size == 0 && (!clip || reinterpret_cast<uintptr_t>(it.out) % size == 0),
                 MOLT_E_VALUE, "%s: gradient %d is not aligned to its type", who, k);
    chunks += (it.count + kChunk - 1) / kChunk;
  }
  MOLT_REQUIRE(chunks < (1LL << 31), MOLT_E_CAPABILITY, "%s: more than 2^44 elements", who);
  return MOLT_OK;
}

// No output may be read as another gradient or written twice: sorted by address, the spans written must stand alone,
// but for an item's own gradient under its own output.
int check_overlap(const char* who, const molt_grad_item* items, int count) try {
  std::vector<Span> spans;
  spans.reserve((size_t)count * 2);
  for (int k = 0; k < count; ++k) {
    const uintptr_t bytes = (uintptr_t)items[k].count * (items[k].dtype == MOLT_DTYPE_BF16 ? 2 : 4);
    if (bytes == 0) continue;
    const uintptr_t g = reinterpret_cast<uintptr_t>(items[k].grad), o = reinterpret_cast<uintptr_t>(items[k].out);
    spans.push_back({o, o + bytes, k, true});
    if (g != o) spans.push_back({g, g + bytes, k, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t read_end = 0, write_end = 0;
  for (const Span& s : spans) {
    MOLT_REQUIRE(s.begin >= write_end && (!s.written || s.begin >= read_end), MOLT_E_VALUE,
                 "%s: the output of one gradient overlaps another gradient or output (item %d)", who, s.item);
    (s.written ? write_end : read_end) = std::max(s.written ? write_end : read_end, s.end);
  }
  return MOLT_OK;
} catch (...) {   // no exception leaves through the C interface
  return fail(MOLT_E_RUNTIME, "%s: out of host memory", who);
}

int norm_launch(const char* who, const molt_grad_item* items, int count, int norm_kind, float grad_scale, float max_norm,
                float* result, void* workspace, size_t workspace_bytes, bool clip, cudaStream_t s) {
  if (int rc = check_items(who, items, count, clip)) return rc;
  MOLT_REQUIRE(norm_kind == MOLT_NORM_L2 || norm_kind == MOLT_NORM_MAX, MOLT_E_VALUE, "%s: unknown norm %d", who, norm_kind);
  MOLT_REQUIRE(max_norm >= 0.f && !isnan(grad_scale), MOLT_E_VALUE, "%s: max_norm must not be negative", who);
  MOLT_REQUIRE(result && workspace && workspace_bytes >= molt_grad_norm_workspace_bytes(count) &&
                   reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
               MOLT_E_VALUE, "%s: the workspace is too small or not 8-byte aligned", who);
  if (clip)
    if (int rc = check_overlap(who, items, count)) return rc;
  auto* part = reinterpret_cast<double*>(workspace);
  const bool max = norm_kind == MOLT_NORM_MAX;
  int parts = 0;
  for (int t = 0; t < tables_of(count); ++t) {
    const molt_grad_item* first = items + t * kTable;
    const int n = std::min(kTable, count - t * kTable), blocks = blocks_for(first, n, kBlocks);
    if (int rc = max ? launch_norm<true>(first, n, blocks, part + parts, s) : launch_norm<false>(first, n, blocks, part + parts, s))
      return rc;
    parts += blocks;
  }
  if (!clip) {
    launch_behind(max ? norm_finish_kernel<true> : norm_finish_kernel<false>, 1, kThreads, s, part, parts, grad_scale, max_norm, result);
    return launch_status("norm_finish_kernel");
  }
  for (int t = tables_of(count) - 1; t >= 0; --t) {
    const molt_grad_item* first = items + t * kTable;
    const int n = std::min(kTable, count - t * kTable), blocks = blocks_for(first, n, kScaleBlocks);
    if (int rc = max ? launch_scale<true>(first, n, blocks, part, parts, max_norm, result, s)
                     : launch_scale<false>(first, n, blocks, part, parts, max_norm, result, s))
      return rc;
  }
  return MOLT_OK;
}

}  // namespace
}  // namespace molt

using namespace molt;

extern "C" size_t molt_grad_norm_workspace_bytes(int count) {
  return count <= 0 ? 0 : (size_t)tables_of(count) * kBlocks * sizeof(double);
}

extern "C" int molt_grad_norm(const molt_grad_item* items, int count, int norm_kind, float grad_scale, float max_norm,
                              float* result, void* workspace, size_t workspace_bytes, uintptr_t stream) {
  return norm_launch("molt_grad_norm", items, count, norm_kind, grad_scale, max_norm, result, workspace, workspace_bytes, false,
                     reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int molt_clip_grads(const molt_grad_item* items, int count, int norm_kind, float max_norm, float* result,
                               void* workspace, size_t workspace_bytes, uintptr_t stream) {
  return norm_launch("molt_clip_grads", items, count, norm_kind, 1.f, max_norm, result, workspace, workspace_bytes, true,
                     reinterpret_cast<cudaStream_t>(stream));
}

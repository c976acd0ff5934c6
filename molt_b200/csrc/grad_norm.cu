// Global norm of a list of gradients, the clipping coefficient, and the clipped gradients.
//   norm = (sum g^2)^(1/2)  or  max |g|;   coefficient = min(1, max_norm / (norm + 1e-6));   out = g * coefficient
// The list travels in the kernel's parameters (no copy to the device, nothing kept, capture-safe); a list longer than a
// table is walked in several launches.  Every tensor is cut into chunks, the chunks of the list are numbered through, and
// block i of G takes chunks i, i + G, ...; it leaves one partial sum, and the partial sums are added in their order, so a list
// gives the same bits on every call.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.cuh"

namespace molt {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 512;          // tensors per launch: the table must stay below the 32764 bytes of kernel parameters
constexpr int kChunk = 8192;         // elements of a chunk
constexpr int kBlocks = 148 * 4;     // a fixed figure: it decides which chunks one partial sum holds

struct Table {
  const void* grad[kTable];
  void* out[kTable];
  long long elements[kTable];
  unsigned first[kTable + 1];        // number of a tensor's first chunk; [count] = all chunks
  unsigned char half[kTable];        // bf16
  int count;
};
static_assert(sizeof(Table) < 32000, "kernel parameters");

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
  if (threadIdx.x == 0)
    for (int w = 1; w < warps; ++w) v = MAX ? larger(v, part[w]) : v + part[w];
  __syncthreads();
  return v;
}

// The tensor that chunk `c` belongs to.
__device__ __forceinline__ int tensor_of(const Table& table, unsigned c) {
  int low = 0, high = table.count - 1;
  while (low < high) {
    const int middle = (low + high + 1) >> 1;
    if (table.first[middle] <= c) low = middle;
    else high = middle - 1;
  }
  return low;
}

template <bool MAX, typename T>
__device__ __forceinline__ double chunk_total(const T* g, int n, double acc) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const double v = load1(g + i);
    acc = MAX ? larger(acc, fabs(v)) : acc + v * v;
  }
  return acc;
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Table table, double* __restrict__ part) {
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

template <bool MAX>
__global__ void __launch_bounds__(1024) norm_finish_kernel(const double* __restrict__ part, int parts, float grad_scale,
                                                           float max_norm, float* __restrict__ result) {
  double acc = 0.;
  for (int i = threadIdx.x; i < parts; i += blockDim.x) acc = MAX ? larger(acc, part[i]) : acc + part[i];
  acc = block_total<MAX>(acc);
  if (threadIdx.x == 0) {
    const float norm = (float)((MAX ? acc : sqrt(acc)) * fabs((double)grad_scale));
    const float c = max_norm / (norm + 1e-6f);
    result[0] = norm;
    result[1] = c > 1.f ? 1.f : c;   // NaN stays
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* g, T* out, int n, float c) {
  for (int i = threadIdx.x; i < n; i += kThreads) store1(out + i, load1(g + i) * c);
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table table, const float* __restrict__ result) {
  const float coefficient = result[1];
  const unsigned chunks = table.first[table.count];
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int k = tensor_of(table, c);
    const long long begin = (long long)(c - table.first[k]) * kChunk;
    const int n = (int)min((long long)kChunk, table.elements[k] - begin);
    if (table.half[k])
      chunk_scale(reinterpret_cast<const __nv_bfloat16*>(table.grad[k]) + begin,
                  reinterpret_cast<__nv_bfloat16*>(table.out[k]) + begin, n, coefficient);
    else
      chunk_scale(reinterpret_cast<const float*>(table.grad[k]) + begin, reinterpret_cast<float*>(table.out[k]) + begin, n,
                  coefficient);
  }
}

int tables_of(int count) { return (count + kTable - 1) / kTable; }

// Fills `table` with items [begin, begin + n).
void fill(Table& table, const molt_grad_item* items, int n) {
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
  Table table;
  for (int t = 0; t < tables_of(count); ++t) {
    fill(table, items + t * kTable, std::min(kTable, count - t * kTable));
    if (norm_kind == MOLT_NORM_MAX) norm_kernel<true><<<kBlocks, kThreads, 0, s>>>(table, part + t * kBlocks);
    else norm_kernel<false><<<kBlocks, kThreads, 0, s>>>(table, part + t * kBlocks);
    if (int rc = launch_status("norm_kernel")) return rc;
  }
  const int parts = tables_of(count) * kBlocks;
  if (norm_kind == MOLT_NORM_MAX) norm_finish_kernel<true><<<1, 1024, 0, s>>>(part, parts, grad_scale, max_norm, result);
  else norm_finish_kernel<false><<<1, 1024, 0, s>>>(part, parts, grad_scale, max_norm, result);
  if (int rc = launch_status("norm_finish_kernel")) return rc;
  if (!clip) return MOLT_OK;
  for (int t = 0; t < tables_of(count); ++t) {
    fill(table, items + t * kTable, std::min(kTable, count - t * kTable));
    scale_kernel<<<kBlocks, kThreads, 0, s>>>(table, result);
    if (int rc = launch_status("scale_kernel")) return rc;
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

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

// The running pair (maximum m, sum s of exp2((x - m) c)) of two parts joined.  A part without a finite logit has m = -inf
// and s = 0; NaN logits leave NaN in s.
__device__ __forceinline__ void join(float& m, float& s, float om, float os, float c) {
  const float nm = fmaxf(m, om);
  const float a = m == nm ? s : s * exp2f((m - nm) * c);
  const float b = om == nm ? os : os * exp2f((om - nm) * c);
  m = nm;
  s = a + b;
}

constexpr int kThreads = 512;

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads) row_kernel(const T* logits, long long row_stride, const long long* __restrict__ ids,
                                                       const float* __restrict__ weight, float inv_t, float* __restrict__ logprob,
                                                       float2* __restrict__ stats, T* grad, long long grad_stride, int vocab) {
  __shared__ float part_m[kThreads / 32], part_s[kThreads / 32];
  const long long row = blockIdx.x, t = ids[row];
  const T* x = logits + row * row_stride;
  T* g = GRAD ? grad + row * grad_stride : nullptr;
  if (t < 0 || t >= vocab) {
    if (threadIdx.x == 0) {
      logprob[row] = 0.f;
      if (stats != nullptr) stats[row] = make_float2(0.f, 0.f);
    }
    if (GRAD)
      for (int v = threadIdx.x; v < vocab; v += kThreads) store1(g + v, 0.f);
    return;
  }
  const float c = inv_t * kLog2e;
  float m = -INFINITY, s = 0.f;
  for (int v = threadIdx.x; v < vocab; v += kThreads) {
    const float xv = load1(x + v);
    if (xv == -INFINITY) continue;   // probability zero
    join(m, s, xv, 1.f, c);
    if (isnan(xv)) s = xv;
  }
  const float xt = load1(x + t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), c);
  if ((threadIdx.x & 31) == 0) {
    part_m[threadIdx.x >> 5] = m;
    part_s[threadIdx.x >> 5] = s;
  }
  __syncthreads();
  m = part_m[0];
  s = part_s[0];
  for (int w = 1; w < kThreads / 32; ++w) join(m, s, part_m[w], part_s[w], c);
  if (m == INFINITY) s = NAN;
  const float log2_s = log2f(s);
  const float l = (xt - m) * inv_t - log2_s * kLn2;
  if (threadIdx.x == 0) {
    logprob[row] = l;
    if (stats != nullptr) stats[row] = make_float2(m, log2_s);
  }
  if (GRAD) {
    const float w = (weight != nullptr ? weight[row] : 1.f) * inv_t;
    __syncthreads();   // the target's logit has been read by all before it may be overwritten
    for (int v = threadIdx.x; v < vocab; v += kThreads)
      store1(g + v, v == t ? -expm1f(l) * w : -exp2f((load1(x + v) - m) * c - log2_s) * w);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) backward_kernel(const T* logits, long long row_stride,
                                                            const long long* __restrict__ ids,
                                                            const float2* __restrict__ stats,
                                                            const float* __restrict__ grad_logprob, float inv_t, T* grad,
                                                            long long grad_stride, int vocab) {
  const long long row = blockIdx.x, t = ids[row];
  const T* x = logits + row * row_stride;
  T* g = grad + row * grad_stride;
  if (t < 0 || t >= vocab) {
    for (int v = threadIdx.x; v < vocab; v += kThreads) store1(g + v, 0.f);
    return;
  }
  const float c = inv_t * kLog2e, m = stats[row].x, log2_s = stats[row].y;
  const float w = grad_logprob[row] * inv_t;
  for (int v = threadIdx.x; v < vocab; v += kThreads) {
    const float d = load1(x + v) - m;
    store1(g + v, v == t ? -expm1f(d * inv_t - log2_s * kLn2) * w : -exp2f(d * c - log2_s) * w);
  }
}

int check_rows(const char* who, const void* logits, int dtype, int64_t row_stride, const int64_t* ids, float temperature,
               int64_t rows, int64_t vocab) {
  MOLT_REQUIRE(rows >= 0 && vocab > 0, MOLT_E_VALUE, "%s: bad shape", who);
  MOLT_REQUIRE(rows <= (1LL << 27) && vocab <= (1LL << 30), MOLT_E_CAPABILITY, "%s: more than 2^27 rows or 2^30 columns", who);
  MOLT_REQUIRE(dtype == MOLT_DTYPE_BF16 || dtype == MOLT_DTYPE_F32, MOLT_E_CAPABILITY, "%s: logits must be bf16 or fp32", who);
  MOLT_REQUIRE(temperature > 0.f && isfinite(temperature) && isfinite(1.f / temperature), MOLT_E_VALUE,
               "%s: temperature must be positive and finite", who);
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logits && ids, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  MOLT_REQUIRE(row_stride == 0 || row_stride >= vocab, MOLT_E_VALUE, "%s: rows of logits overlap", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == MOLT_DTYPE_BF16 ? 2 : 4) == 0, MOLT_E_VALUE,
               "%s: logits are not aligned to their type", who);
  return MOLT_OK;
}

// The gradient may lie over the logits exactly, or beside them (also in other columns of the same wider rows).
int check_grad(const char* who, const void* logits, int dtype, int64_t row_stride, const void* grad, int64_t grad_stride,
               int64_t rows, int64_t vocab) {
  if (rows == 0) return MOLT_OK;
  const int64_t size = dtype == MOLT_DTYPE_BF16 ? 2 : 4;
  MOLT_REQUIRE(grad != nullptr, MOLT_E_VALUE, "%s: NULL gradient pointer", who);
  MOLT_REQUIRE(reinterpret_cast<uintptr_t>(grad) % size == 0, MOLT_E_VALUE, "%s: the gradient is not aligned to its type", who);
  MOLT_REQUIRE(grad_stride >= vocab, MOLT_E_VALUE, "%s: rows of the gradient overlap", who);
  const intptr_t a = reinterpret_cast<intptr_t>(logits), b = reinterpret_cast<intptr_t>(grad);
  if (a == b && (row_stride == grad_stride || rows == 1)) return MOLT_OK;
  const intptr_t a_end = a + ((rows - 1) * row_stride + vocab) * size, b_end = b + ((rows - 1) * grad_stride + vocab) * size;
  if (a_end <= b || b_end <= a) return MOLT_OK;
  if (row_stride == grad_stride) {
    const intptr_t pitch = row_stride * size, shift = (((b - a) % pitch) + pitch) % pitch;
    if (shift >= vocab * size && shift <= pitch - vocab * size) return MOLT_OK;
  }
  return fail(MOLT_E_VALUE, "%s: the gradient overlaps the logits without being the same rows", who);
}

template <typename T>
int launch_rows(const void* logits, int64_t row_stride, const int64_t* ids, const float* weight, float temperature,
                float* logprob, float* stats, void* grad, int64_t grad_stride, int64_t rows, int64_t vocab, cudaStream_t s) {
  auto* x = reinterpret_cast<const T*>(logits);
  auto* id = reinterpret_cast<const long long*>(ids);
  auto* st = reinterpret_cast<float2*>(stats);
  if (grad != nullptr)
    row_kernel<T, true><<<(unsigned)rows, kThreads, 0, s>>>(x, row_stride, id, weight, 1.f / temperature, logprob, st,
                                                            reinterpret_cast<T*>(grad), grad_stride, (int)vocab);
  else
    row_kernel<T, false><<<(unsigned)rows, kThreads, 0, s>>>(x, row_stride, id, weight, 1.f / temperature, logprob, st, nullptr, 0,
                                                             (int)vocab);
  return launch_status("token_logprob row_kernel");
}

}  // namespace
}  // namespace molt

using namespace molt;

extern "C" int molt_token_logprob_fwd(const void* logits, int dtype, int64_t row_stride, const int64_t* token_ids,
                                      float temperature, float* logprob, float* stats, int64_t rows, int64_t vocab,
                                      uintptr_t stream) {
  if (int rc = check_rows("molt_token_logprob_fwd", logits, dtype, row_stride, token_ids, temperature, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logprob != nullptr, MOLT_E_VALUE, "molt_token_logprob_fwd: NULL tensor pointer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MOLT_DTYPE_BF16
             ? launch_rows<__nv_bfloat16>(logits, row_stride, token_ids, nullptr, temperature, logprob, stats, nullptr, 0, rows, vocab, s)
             : launch_rows<float>(logits, row_stride, token_ids, nullptr, temperature, logprob, stats, nullptr, 0, rows, vocab, s);
}

extern "C" int molt_token_logprob_grad(const void* logits, int dtype, int64_t row_stride, const int64_t* token_ids,
                                       const float* weight, float temperature, float* logprob, void* grad_logits,
                                       int64_t grad_stride, int64_t rows, int64_t vocab, uintptr_t stream) {
  const char* who = "molt_token_logprob_grad";
  if (int rc = check_rows(who, logits, dtype, row_stride, token_ids, temperature, rows, vocab)) return rc;
  if (int rc = check_grad(who, logits, dtype, row_stride, grad_logits, grad_stride, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(logprob != nullptr, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == MOLT_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(logits, row_stride, token_ids, weight, temperature, logprob, nullptr,
                                                               grad_logits, grad_stride, rows, vocab, s)
                                  : launch_rows<float>(logits, row_stride, token_ids, weight, temperature, logprob, nullptr,
                                                       grad_logits, grad_stride, rows, vocab, s);
}

extern "C" int molt_token_logprob_bwd(const void* logits, int dtype, int64_t row_stride, const int64_t* token_ids,
                                      const float* stats, const float* grad_logprob, float temperature, void* grad_logits,
                                      int64_t grad_stride, int64_t rows, int64_t vocab, uintptr_t stream) {
  const char* who = "molt_token_logprob_bwd";
  if (int rc = check_rows(who, logits, dtype, row_stride, token_ids, temperature, rows, vocab)) return rc;
  if (int rc = check_grad(who, logits, dtype, row_stride, grad_logits, grad_stride, rows, vocab)) return rc;
  if (rows == 0) return MOLT_OK;
  MOLT_REQUIRE(stats && grad_logprob, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* id = reinterpret_cast<const long long*>(token_ids);
  auto* st = reinterpret_cast<const float2*>(stats);
  if (dtype == MOLT_DTYPE_BF16)
    backward_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, s>>>(
        reinterpret_cast<const __nv_bfloat16*>(logits), row_stride, id, st, grad_logprob, 1.f / temperature,
        reinterpret_cast<__nv_bfloat16*>(grad_logits), grad_stride, (int)vocab);
  else
    backward_kernel<float><<<(unsigned)rows, kThreads, 0, s>>>(reinterpret_cast<const float*>(logits), row_stride, id, st,
                                                               grad_logprob, 1.f / temperature,
                                                               reinterpret_cast<float*>(grad_logits), grad_stride, (int)vocab);
  return launch_status("token_logprob backward_kernel");
}

// Losses over token log-probabilities: the clipped policy loss with a KL term, and the loss over preference pairs.
// All of it is one pass over a few fp32 arrays of [batch, seq] (HBM- or, for small batches, launch-bound).  The weights
// of the mean are only known once all masks have been counted, and the scale of the gradient arrives with the backward
// pass, so the forward writes the gradient without either and the backward multiplies both in.
#include <math.h>

#include "common.cuh"

namespace molt {
namespace {

constexpr int kThreads = 256;

// Sum over a block in a fixed order; the result is valid in thread 0.
template <int N>
__device__ __forceinline__ void block_sum(double (&v)[N]) {
  __shared__ double part[N][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(~0u, v[i], o);
    if (lane == 0) part[i][warp] = v[i];
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 0; i < N; ++i) {
      double sum = 0.;
      for (int w = 0; w < warps; ++w) sum += part[i][w];
      v[i] = sum;
    }
  __syncthreads();
}

// Tokens of a row one block takes: a row is cut when there are fewer rows than the device has room for blocks.
int splits_for(int64_t rows, int64_t seq) {
  const int64_t most = (seq + kThreads * 4 - 1) / (kThreads * 4);
  int64_t want = ((int64_t)148 * 8 + rows - 1) / rows;   // a fixed figure: the split decides the order of the sums
  if (want > most) want = most;
  return (int)(want < 1 ? 1 : want > 1024 ? 1024 : want);
}

// A batch this small is one block's work: its row sums stay in shared memory and one launch gives the loss (4 x 64 tokens,
// whole call with its backward: 135 us of host time with two launches and a workspace, 113 us with one).
constexpr int kOneBlock = 1024, kOneBlockRows = 256, kOneBlockTokens = 8192;
bool one_block(int64_t rows, int64_t seq) { return rows <= kOneBlockRows && rows * seq <= kOneBlockTokens; }
// Warps of the one block that share a row.
int one_block_splits(int64_t rows) { return rows >= kOneBlock / 32 ? 1 : (int)(kOneBlock / 32 / rows); }

// ---- clipped policy loss -------------------------------------------------------------------------------------------
struct PolicyArgs {
  const float *logprob, *old, *ref, *advantage;
  const uint8_t* mask;
  long long lp_stride, old_stride, ref_stride, adv_stride, mask_stride;
  long long batch, seq;
  int per_token, splits;
  double log_high, log_low;   // ln(1 + clip_high), ln(1 - clip_low): the borders of ln r
  float log_high_f, log_low_f, high, low, kl_coef;   // the borders rounded to fp32; 1 + clip_high, 1 - clip_low
};

// exp(d) - 1 - d without the cancellation: the Taylor series d^2/2 (1 + d/3 (1 + d/4 (...))) where |d| is small (its
// truncation is below 2^-26 relative for |d| <= 0.5 with ten terms), the plain difference elsewhere.
__device__ __forceinline__ float exp_minus_1_minus(float d) {
  if (d > 60.f) return expf(d);   // 1 + d is below its last bit; an infinite d must not meet itself
  if (fabsf(d) > 0.5f) return expm1f(d) - d;
  float r = 1.f;
#pragma unroll
  for (int k = 10; k >= 3; --k) r = fmaf(r, d * (1.f / k), 1.f);
  return 0.5f * d * d * r;
}

// Tokens begin, begin + step, ... below end of row b, kUnroll of them loaded at a time.
constexpr int kUnroll = 4;

__device__ __forceinline__ void policy_tokens(const PolicyArgs& a, long long b, long long begin, long long end, int step,
                                              float* __restrict__ unit_grad, double (&sum)[4]) {
  for (long long t0 = begin; t0 < end; t0 += kUnroll * step) {
    float lp[kUnroll], old[kUnroll], adv[kUnroll], ref[kUnroll];
    bool kept[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long t = t0 + j * step;
      kept[j] = t < end;
      if (kept[j]) {
        lp[j] = a.logprob[b * a.lp_stride + t];
        old[j] = a.old[b * a.old_stride + t];
        adv[j] = a.advantage[b * a.adv_stride + (a.per_token ? t : 0)];
        ref[j] = a.ref != nullptr ? a.ref[b * a.ref_stride + t] : 0.f;
        kept[j] = a.mask == nullptr || a.mask[b * a.mask_stride + t] != 0;
      }
    }
    float loss = 0.f, ks = 0.f;
    int cuts = 0, keeps = 0;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      float g = 0.f;
      if (kept[j]) {
        // fp32 rounds monotonously, so the rounded difference decides the border unless it lies on it
        const float d = lp[j] - old[j];
        bool cut = (adv[j] > 0.f && d > a.log_high_f) || (adv[j] < 0.f && d < a.log_low_f);
        if (d == a.log_high_f || d == a.log_low_f) {
          const double exact = (double)lp[j] - (double)old[j];
          cut = (adv[j] > 0.f && exact > a.log_high) || (adv[j] < 0.f && exact < a.log_low);
        }
        float l = 0.f;
        if (adv[j] != 0.f) {   // the product with an advantage of zero is zero however large the ratio (NaN stays NaN)
          const float r = expf(d);
          l = -(cut ? (adv[j] > 0.f ? a.high : a.low) : r) * adv[j];
          g = cut ? 0.f : -r * adv[j];
        }
        if (a.ref != nullptr) {
          const float e = ref[j] - lp[j], k = exp_minus_1_minus(e);
          l += a.kl_coef * k;
          g -= a.kl_coef * (k + e);   // exp(e) - 1
          ks += k;
        }
        loss += l;
        cuts += cut;
        ++keeps;
      }
      if (unit_grad != nullptr && t0 + j * step < end) unit_grad[b * a.seq + t0 + j * step] = g;
    }
    // four tokens in fp32, then in 64 bits: three roundings more on values that carry a few already
    sum[0] += loss;
    sum[1] += ks;
    sum[2] += cuts;
    sum[3] += keeps;
  }
}

// Row sums (loss, k, cut, kept), weights and the result, by one block.
__device__ __forceinline__ void policy_finish(const double* part, long long batch, int splits, int reduction,
                                              float* __restrict__ row_weight, float* __restrict__ loss,
                                              float* __restrict__ stats) {
  __shared__ double total;
  const auto row_sum = [&](long long b, double (&row)[4]) {
    for (int i = 0; i < 4; ++i) row[i] = 0.;
    for (int s = 0; s < splits; ++s)
      for (int i = 0; i < 4; ++i) row[i] += part[(b * splits + s) * 4 + i];
  };
  // a thread's first row is read once; rows beyond the block's size a second time
  double first[4] = {0., 0., 0., 0.}, row[4];
  double count[1] = {0.};
  for (long long b = threadIdx.x; b < batch; b += blockDim.x) {
    row_sum(b, row);
    if (b < blockDim.x)
      for (int i = 0; i < 4; ++i) first[i] = row[i];
    count[0] += reduction == MOLT_REDUCE_TOKEN ? row[3] : (row[3] > 0. ? 1. : 0.);
  }
  block_sum(count);
  if (threadIdx.x == 0) total = count[0];
  __syncthreads();
  double sum[3] = {0., 0., 0.};
  for (long long b = threadIdx.x; b < batch; b += blockDim.x) {
    if (b < blockDim.x) {
      for (int i = 0; i < 4; ++i) row[i] = first[i];
    } else {
      row_sum(b, row);
    }
    double w = 0.;
    if (row[3] > 0.) {
      w = reduction == MOLT_REDUCE_TOKEN ? 1. / total : 1. / (total * row[3]);
      for (int i = 0; i < 3; ++i) sum[i] += w * row[i];
    }
    if (row_weight != nullptr) row_weight[b] = (float)w;
  }
  block_sum(sum);
  if (threadIdx.x == 0) {
    loss[0] = (float)sum[0];
    stats[0] = (float)sum[1];
    stats[1] = (float)sum[2];
  }
}

__global__ void __launch_bounds__(kThreads) policy_kernel(PolicyArgs a, float* __restrict__ unit_grad, double* __restrict__ part) {
  const long long b = blockIdx.x;
  const long long begin = a.seq * blockIdx.y / a.splits, end = a.seq * (blockIdx.y + 1) / a.splits;
  double sum[4] = {0., 0., 0., 0.};
  policy_tokens(a, b, begin + threadIdx.x, end, kThreads, unit_grad, sum);
  block_sum(sum);
  if (threadIdx.x == 0)
    for (int i = 0; i < 4; ++i) part[(b * a.splits + blockIdx.y) * 4 + i] = sum[i];
}

__global__ void __launch_bounds__(1024) policy_finish_kernel(const double* __restrict__ part, long long batch, int splits,
                                                             int reduction, float* __restrict__ row_weight,
                                                             float* __restrict__ loss, float* __restrict__ stats) {
  policy_finish(part, batch, splits, reduction, row_weight, loss, stats);
}

// The whole forward in one block: a warp takes one of the splits of a row.
__global__ void __launch_bounds__(kOneBlock) policy_one_block_kernel(PolicyArgs a, int reduction, float* __restrict__ unit_grad,
                                                                     float* __restrict__ row_weight, float* __restrict__ loss,
                                                                     float* __restrict__ stats) {
  __shared__ double part[kOneBlockRows * 4];
  const int lane = threadIdx.x & 31, units = (int)a.batch * a.splits;
  for (int u = threadIdx.x >> 5; u < units; u += kOneBlock / 32) {
    const int b = u / a.splits, s = u - b * a.splits;
    double sum[4] = {0., 0., 0., 0.};
    policy_tokens(a, b, a.seq * s / a.splits + lane, a.seq * (s + 1) / a.splits, 32, unit_grad, sum);
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(~0u, sum[i], o);
      if (lane == 0) part[u * 4 + i] = sum[i];
    }
  }
  __syncthreads();
  policy_finish(part, a.batch, a.splits, reduction, row_weight, loss, stats);
}

// Backward passes: a thread takes kUnroll tokens of one row, so that a block is one round of loads and stores.
constexpr int kBackTokens = kThreads * kUnroll;

__global__ void __launch_bounds__(kThreads) policy_backward_kernel(const float* __restrict__ unit_grad,
                                                                   const float* __restrict__ row_weight,
                                                                   const float* __restrict__ grad_loss,
                                                                   float* __restrict__ grad_logprob, long long seq) {
  const long long b = blockIdx.x, first = b * seq, t0 = (long long)blockIdx.y * kBackTokens + threadIdx.x;
  float u[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) u[j] = t0 + j * kThreads < seq ? unit_grad[first + t0 + j * kThreads] : 0.f;
  const float w = row_weight[b] * grad_loss[0];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j)
    if (t0 + j * kThreads < seq) grad_logprob[first + t0 + j * kThreads] = u[j] == 0.f ? 0.f : u[j] * w;
}

// ---- preference pairs ----------------------------------------------------------------------------------------------
struct PreferenceArgs {
  const float *logprob, *ref;
  const uint8_t* mask;
  long long lp_stride, ref_stride, mask_stride;
  long long pairs, seq;
  int ref_per_token, splits, kind, average;
  double beta, smoothing;
};

__device__ __forceinline__ void preference_tokens(const PreferenceArgs& a, long long i, long long begin, long long end, int step,
                                                  double (&sum)[2]) {
  int keeps = 0;
  for (long long t0 = begin; t0 < end; t0 += kUnroll * step) {
    float lp[kUnroll], ref[kUnroll];
    bool kept[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const long long t = t0 + j * step;
      kept[j] = t < end;
      if (kept[j]) {
        lp[j] = a.logprob[i * a.lp_stride + t];
        ref[j] = a.ref != nullptr && a.ref_per_token ? a.ref[i * a.ref_stride + t] : 0.f;
        kept[j] = a.mask == nullptr || a.mask[i * a.mask_stride + t] != 0;
      }
    }
#pragma unroll
    for (int j = 0; j < kUnroll; j += 2) {
      // a pair of fp32 differences is added before it goes on in 64 bits: two roundings of the terms' magnitudes
      const float d0 = kept[j] ? lp[j] - ref[j] : 0.f, d1 = kept[j + 1] ? lp[j + 1] - ref[j + 1] : 0.f;
      sum[0] += d0 + d1;
      keeps += (int)kept[j] + (int)kept[j + 1];
    }
  }
  sum[1] += keeps;
}

__device__ __forceinline__ void preference_finish(const PreferenceArgs& a, const double* part, float* __restrict__ seq_grad,
                                                  float* __restrict__ rewards, float* __restrict__ loss_out) {
  double total[1] = {0.};
  for (long long p = threadIdx.x; p < a.pairs; p += blockDim.x) {
    double s[2], scale[2];
    for (int side = 0; side < 2; ++side) {
      const long long i = p + side * a.pairs;
      double sum = 0., kept = 0.;
      for (int k = 0; k < a.splits; ++k) {
        sum += part[(i * a.splits + k) * 2];
        kept += part[(i * a.splits + k) * 2 + 1];
      }
      scale[side] = a.average ? (kept > 0. ? 1. / kept : 0.) : 1.;
      s[side] = a.average ? (kept > 0. ? sum / kept : 0.) : sum;
      if (a.ref != nullptr && !a.ref_per_token) s[side] -= (double)a.ref[i * a.ref_stride];
      rewards[i] = (float)(a.beta * s[side]);
    }
    const double h = s[0] - s[1];
    double loss, slope;
    if (a.kind == MOLT_PREFERENCE_SIGMOID) {
      const double z = a.beta * h, e = exp(-fabs(z)), soft = log1p(e);   // -ln sig(z) = soft + max(-z, 0)
      loss = soft + (1. - a.smoothing) * fmax(-z, 0.) + a.smoothing * fmax(z, 0.);
      if (isnan(z)) loss = z;
      const double small = e / (1. + e), large = 1. / (1. + e);          // sig(-|z|), sig(|z|)
      slope = -a.beta * ((1. - a.smoothing) * (z >= 0. ? small : large) - a.smoothing * (z >= 0. ? large : small));
    } else if (a.kind == MOLT_PREFERENCE_HINGE) {
      const double z = 1. - a.beta * h;
      loss = z > 0. ? z : (isnan(z) ? z : 0.);
      slope = isnan(z) ? z : (a.beta * h < 1. ? -a.beta : 0.);
    } else {
      const double z = h - 1. / (2. * a.beta);
      loss = z * z;
      slope = 2. * z;
    }
    total[0] += loss / (double)a.pairs;
    if (seq_grad != nullptr) {
      seq_grad[p] = (float)(slope * scale[0] / (double)a.pairs);
      seq_grad[p + a.pairs] = (float)(-slope * scale[1] / (double)a.pairs);
    }
  }
  block_sum(total);
  if (threadIdx.x == 0) loss_out[0] = (float)total[0];
}

__global__ void __launch_bounds__(kThreads) preference_kernel(PreferenceArgs a, double* __restrict__ part) {
  const long long i = blockIdx.x;
  const long long begin = a.seq * blockIdx.y / a.splits, end = a.seq * (blockIdx.y + 1) / a.splits;
  double sum[2] = {0., 0.};
  preference_tokens(a, i, begin + threadIdx.x, end, kThreads, sum);
  block_sum(sum);
  if (threadIdx.x == 0) {
    part[(i * a.splits + blockIdx.y) * 2] = sum[0];
    part[(i * a.splits + blockIdx.y) * 2 + 1] = sum[1];
  }
}

__global__ void __launch_bounds__(1024) preference_finish_kernel(PreferenceArgs a, const double* __restrict__ part,
                                                                 float* __restrict__ seq_grad, float* __restrict__ rewards,
                                                                 float* __restrict__ loss) {
  preference_finish(a, part, seq_grad, rewards, loss);
}

__global__ void __launch_bounds__(kOneBlock) preference_one_block_kernel(PreferenceArgs a, float* __restrict__ seq_grad,
                                                                         float* __restrict__ rewards, float* __restrict__ loss) {
  __shared__ double part[kOneBlockRows * 2];
  const int lane = threadIdx.x & 31, units = (int)(2 * a.pairs) * a.splits;
  for (int u = threadIdx.x >> 5; u < units; u += kOneBlock / 32) {
    const int i = u / a.splits, s = u - i * a.splits;
    double sum[2] = {0., 0.};
    preference_tokens(a, i, a.seq * s / a.splits + lane, a.seq * (s + 1) / a.splits, 32, sum);
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[k] += __shfl_xor_sync(~0u, sum[k], o);
      if (lane == 0) part[u * 2 + k] = sum[k];
    }
  }
  __syncthreads();
  preference_finish(a, part, seq_grad, rewards, loss);
}

__global__ void __launch_bounds__(kThreads) preference_backward_kernel(const uint8_t* __restrict__ mask, long long mask_stride,
                                                                       const float* __restrict__ seq_grad,
                                                                       const float* __restrict__ grad_loss,
                                                                       float* __restrict__ grad_logprob, long long seq) {
  const long long i = blockIdx.x, t0 = (long long)blockIdx.y * kBackTokens + threadIdx.x;
  bool kept[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j)
    kept[j] = t0 + j * kThreads < seq && (mask == nullptr || mask[i * mask_stride + t0 + j * kThreads] != 0);
  const float g = seq_grad[i] * grad_loss[0];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j)
    if (t0 + j * kThreads < seq) grad_logprob[i * seq + t0 + j * kThreads] = kept[j] ? g : 0.f;
}

int check_sizes(const char* who, int64_t rows, int64_t seq) {
  MOLT_REQUIRE(rows >= 0 && seq >= 0, MOLT_E_VALUE, "%s: negative size", who);
  MOLT_REQUIRE(rows < (1LL << 31) && seq <= (1LL << 25), MOLT_E_CAPABILITY, "%s: 2^31 sequences or more than 2^25 tokens in one", who);
  return MOLT_OK;
}

int check_stride(const char* who, const char* what, int64_t stride, int64_t least) {
  MOLT_REQUIRE(stride >= least || stride == 0, MOLT_E_VALUE, "%s: rows of %s overlap", who, what);
  return MOLT_OK;
}

}  // namespace
}  // namespace molt

using namespace molt;

extern "C" size_t molt_policy_loss_workspace_bytes(int64_t batch, int64_t seq) {
  if (batch <= 0 || seq < 0 || one_block(batch, seq)) return 0;
  return (size_t)batch * splits_for(batch, seq) * 4 * sizeof(double);
}

extern "C" int molt_policy_loss_fwd(const float* logprob, const float* old_logprob, const float* ref_logprob,
                                    const float* advantage, int advantage_per_token, const uint8_t* mask,
                                    const int64_t row_strides[5], int64_t batch, int64_t seq, double clip_low, double clip_high,
                                    double kl_coef, int reduction, float* unit_grad, float* row_weight, float* loss,
                                    float* stats, void* workspace, size_t workspace_bytes, uintptr_t stream) {
  const char* who = "molt_policy_loss_fwd";
  if (int rc = check_sizes(who, batch, seq)) return rc;
  MOLT_REQUIRE(batch > 0, MOLT_E_VALUE, "%s: no sequence", who);
  MOLT_REQUIRE(reduction == MOLT_REDUCE_TOKEN || reduction == MOLT_REDUCE_SEQUENCE, MOLT_E_VALUE, "%s: unknown reduction %d", who,
               reduction);
  MOLT_REQUIRE(clip_low >= 0. && clip_low <= 1. && clip_high >= 0. && isfinite(clip_high) && isfinite(kl_coef), MOLT_E_VALUE,
               "%s: clip_low must lie in [0, 1], clip_high and kl_coef must be finite, clip_high not negative", who);
  MOLT_REQUIRE(row_strides && loss && stats &&
                   (seq == 0 || (unit_grad == nullptr) == (row_weight == nullptr)),
               MOLT_E_VALUE, "%s: NULL pointer", who);
  MOLT_REQUIRE(seq == 0 || (logprob && old_logprob && advantage), MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  const size_t needed = molt_policy_loss_workspace_bytes(batch, seq);
  MOLT_REQUIRE(needed == 0 || (workspace && workspace_bytes >= needed && reinterpret_cast<uintptr_t>(workspace) % 8 == 0), MOLT_E_VALUE,
               "%s: the workspace is too small or not 8-byte aligned", who);
  const char* names[5] = {"logprob", "old_logprob", "ref_logprob", "advantage", "mask"};
  for (int i = 0; i < 5; ++i)
    if (int rc = check_stride(who, names[i], row_strides[i], i == 3 && !advantage_per_token ? 1 : seq)) return rc;
  PolicyArgs a;
  a.logprob = logprob; a.old = old_logprob; a.ref = ref_logprob; a.advantage = advantage; a.mask = mask;
  a.lp_stride = row_strides[0]; a.old_stride = row_strides[1]; a.ref_stride = row_strides[2]; a.adv_stride = row_strides[3];
  a.mask_stride = row_strides[4];
  a.batch = batch; a.seq = seq; a.per_token = advantage_per_token != 0; a.splits = splits_for(batch, seq);
  a.log_high = log1p(clip_high); a.log_low = log1p(-clip_low);
  a.log_high_f = (float)a.log_high; a.log_low_f = (float)a.log_low;
  a.high = (float)(1. + clip_high); a.low = (float)(1. - clip_low); a.kl_coef = (float)kl_coef;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (needed == 0) {
    a.splits = one_block_splits(batch);
    policy_one_block_kernel<<<1, kOneBlock, 0, s>>>(a, reduction, unit_grad, row_weight, loss, stats);
    return launch_status("policy_one_block_kernel");
  }
  auto* part = reinterpret_cast<double*>(workspace);
  policy_kernel<<<dim3((unsigned)batch, a.splits), kThreads, 0, s>>>(a, unit_grad, part);
  if (int rc = launch_status("policy_kernel")) return rc;
  policy_finish_kernel<<<1, 1024, 0, s>>>(part, batch, a.splits, reduction, row_weight, loss, stats);
  return launch_status("policy_finish_kernel");
}

extern "C" int molt_policy_loss_bwd(const float* unit_grad, const float* row_weight, const float* grad_loss, float* grad_logprob,
                                    int64_t batch, int64_t seq, uintptr_t stream) {
  const char* who = "molt_policy_loss_bwd";
  if (int rc = check_sizes(who, batch, seq)) return rc;
  if (batch == 0 || seq == 0) return MOLT_OK;
  MOLT_REQUIRE(unit_grad && row_weight && grad_loss && grad_logprob, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  const dim3 grid((unsigned)batch, (unsigned)((seq + kBackTokens - 1) / kBackTokens));
  policy_backward_kernel<<<grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(unit_grad, row_weight, grad_loss, grad_logprob,
                                                                                       seq);
  return launch_status("policy_backward_kernel");
}

extern "C" size_t molt_preference_loss_workspace_bytes(int64_t pairs, int64_t seq) {
  if (pairs <= 0 || seq < 0 || one_block(2 * pairs, seq)) return 0;
  return (size_t)pairs * 2 * splits_for(pairs * 2, seq) * 2 * sizeof(double);
}

extern "C" int molt_preference_loss_fwd(const float* logprob, const float* ref_logprob, int ref_per_token, const uint8_t* mask,
                                        const int64_t row_strides[3], int64_t pairs, int64_t seq, double beta, double smoothing,
                                        int kind, int average, float* seq_grad, float* rewards, float* loss, void* workspace,
                                        size_t workspace_bytes, uintptr_t stream) {
  const char* who = "molt_preference_loss_fwd";
  MOLT_REQUIRE(pairs > 0 && pairs < (1LL << 30), MOLT_E_VALUE, "%s: no pair", who);
  if (int rc = check_sizes(who, 2 * pairs, seq)) return rc;
  MOLT_REQUIRE(kind >= MOLT_PREFERENCE_SIGMOID && kind <= MOLT_PREFERENCE_IPO, MOLT_E_VALUE, "%s: unknown kind %d", who, kind);
  MOLT_REQUIRE(beta > 0. && isfinite(beta) && smoothing >= 0. && smoothing <= 1., MOLT_E_VALUE,
               "%s: beta must be positive and finite, the smoothing in [0, 1]", who);
  MOLT_REQUIRE(smoothing == 0. || kind == MOLT_PREFERENCE_SIGMOID, MOLT_E_VALUE, "%s: only the sigmoid loss has label smoothing", who);
  MOLT_REQUIRE(row_strides && rewards && loss && (seq == 0 || logprob), MOLT_E_VALUE, "%s: NULL pointer", who);
  const size_t needed = molt_preference_loss_workspace_bytes(pairs, seq);
  MOLT_REQUIRE(needed == 0 || (workspace && workspace_bytes >= needed && reinterpret_cast<uintptr_t>(workspace) % 8 == 0), MOLT_E_VALUE,
               "%s: the workspace is too small or not 8-byte aligned", who);
  const char* names[3] = {"logprob", "ref_logprob", "mask"};
  for (int i = 0; i < 3; ++i)
    if (int rc = check_stride(who, names[i], row_strides[i], i == 1 && !ref_per_token ? 1 : seq)) return rc;
  PreferenceArgs a;
  a.logprob = logprob; a.ref = ref_logprob; a.mask = mask;
  a.lp_stride = row_strides[0]; a.ref_stride = row_strides[1]; a.mask_stride = row_strides[2];
  a.pairs = pairs; a.seq = seq; a.ref_per_token = ref_per_token != 0; a.splits = splits_for(2 * pairs, seq);
  a.kind = kind; a.average = average != 0; a.beta = beta; a.smoothing = smoothing;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (needed == 0) {
    a.splits = one_block_splits(2 * pairs);
    preference_one_block_kernel<<<1, kOneBlock, 0, s>>>(a, seq_grad, rewards, loss);
    return launch_status("preference_one_block_kernel");
  }
  auto* part = reinterpret_cast<double*>(workspace);
  preference_kernel<<<dim3((unsigned)(2 * pairs), a.splits), kThreads, 0, s>>>(a, part);
  if (int rc = launch_status("preference_kernel")) return rc;
  preference_finish_kernel<<<1, 1024, 0, s>>>(a, part, seq_grad, rewards, loss);
  return launch_status("preference_finish_kernel");
}

extern "C" int molt_preference_loss_bwd(const uint8_t* mask, int64_t mask_stride, const float* seq_grad, const float* grad_loss,
                                        float* grad_logprob, int64_t pairs, int64_t seq, uintptr_t stream) {
  const char* who = "molt_preference_loss_bwd";
  MOLT_REQUIRE(pairs >= 0 && pairs < (1LL << 30), MOLT_E_VALUE, "%s: bad pair count", who);
  if (int rc = check_sizes(who, 2 * pairs, seq)) return rc;
  if (pairs == 0 || seq == 0) return MOLT_OK;
  MOLT_REQUIRE(seq_grad && grad_loss && grad_logprob, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  if (int rc = check_stride(who, "mask", mask_stride, seq)) return rc;
  const dim3 grid((unsigned)(2 * pairs), (unsigned)((seq + kBackTokens - 1) / kBackTokens));
  preference_backward_kernel<<<grid, kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(mask, mask_stride, seq_grad, grad_loss,
                                                                                           grad_logprob, seq);
  return launch_status("preference_backward_kernel");
}

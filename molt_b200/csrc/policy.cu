// Losses over token log-probabilities: the clipped policy loss with a KL term, and the loss over preference pairs.
// One pass over a few fp32 arrays of [batch, seq].  The weights of the mean are only known once all masks have been counted,
// and the scale of the gradient arrives with the backward pass, so the forward writes the gradient without either and the
// backward multiplies both in (29 bytes per token in all with a reference; recomputing in the backward would move 38).
// What bounds them (device time a call, forward alone, calls replayed one behind the other): small batches the launches (one for
// a forward of at most 8192 tokens, policy 5.6 us and preference 4; 3 us for a backward); 512 x 4096 tokens the arithmetic of
// about 125 instructions per token and the latency of one wave of blocks (policy 17 us where the bytes would take 5, preference
// 10 us for twice the tokens); 2048 x 4096 tokens HBM to about a half (policy 40 us, preference 14, backward 9-11); tens of
// thousands of pairs their one finishing block (32768 pairs: 112 us).
#include <math.h>

#include <type_traits>

#include "common.cuh"

namespace molt {
namespace {

constexpr int kThreads = 256, kFinish = 512;

// Sums of one thread: N in 64 bits, and M counts.
template <int N, int M>
struct Sums {
  double v[N] = {};
  int n[M] = {};

  // Sums of the warp, in all its lanes.
  __device__ __forceinline__ void join_warp() {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(~0u, v[i], o);
#pragma unroll
    for (int i = 0; i < M; ++i) n[i] = __reduce_add_sync(~0u, n[i]);
  }
  // The sums as N + M doubles.
  __device__ __forceinline__ void store(double* to, int stride) const {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i * stride] = v[i];
#pragma unroll
    for (int i = 0; i < M; ++i) to[(N + i) * stride] = n[i];
  }
};

// Adds up, over a block and in a fixed order, what `store` left of every warp in part[value][warp]: warp i does value i, and
// its lane 0 returns it.
__device__ __forceinline__ double join_block(const double* part, int values) {
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.;
  if (warp < values) {
    sum = lane < (blockDim.x >> 5) ? part[warp * 32 + lane] : 0.;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  }
  return sum;
}

// Sum over a block in a fixed order, for all its threads.
template <int N>
__device__ __forceinline__ void block_sum(double (&v)[N]) {
  __shared__ double part[N * 32], total[N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(~0u, v[i], o);
    if (lane == 0) part[i * 32 + warp] = v[i];
  }
  const double mine = join_block(part, N);
  if (lane == 0 && warp < N) total[warp] = mine;
  __syncthreads();
  for (int i = 0; i < N; ++i) v[i] = total[i];
}

using Full = std::integral_constant<bool, true>;
using Ragged = std::integral_constant<bool, false>;

constexpr int kUnroll = 4;                      // tokens a thread loads at a time
constexpr int kRound = kThreads * kUnroll;      // tokens a block loads at a time

// A row is cut where there are fewer rows than the device has room for blocks, into parts of whole rounds (so that no
// block ends on a round that is mostly empty).  Fixed figures: the cut decides the order of the sums.
int part_tokens(int64_t rows, int64_t seq) {
  const int64_t want = (148 * 8 + rows - 1) / rows, even = (seq + want - 1) / want;
  return (int)(even <= kRound ? kRound : even / kRound * kRound);
}
int splits_for(int64_t rows, int64_t seq) {
  const int64_t per = part_tokens(rows, seq), splits = (seq + per - 1) / per;
  return (int)(splits < 1 ? 1 : splits);
}

// A batch this small is one block's work: its row sums stay in shared memory and one launch gives the loss (4 x 64 tokens,
// whole call with its backward: 135 us of host time with two launches and a workspace, 113 us with one).
constexpr int kOneBlock = 1024, kOneBlockRows = 256, kOneBlockTokens = 8192;
bool one_block(int64_t rows, int64_t seq) { return rows <= kOneBlockRows && rows * seq <= kOneBlockTokens; }
// Warps of the one block that share a row.
int one_block_splits(int64_t rows) { return rows >= kOneBlock / 32 ? 1 : (int)(kOneBlock / 32 / rows); }

// Many short rows: a warp takes a row, a block eight at a time (16384 x 128 tokens with a block per row: 85 us).
constexpr int kWarpRows = 2048, kWarpTokens = kRound, kWarps = kThreads / 32;
bool warp_rows(int64_t rows, int64_t seq) { return rows >= kWarpRows && seq <= kWarpTokens; }
int warp_row_blocks(int64_t rows) { return (int)((rows + kWarps - 1) / kWarps < 148 * 8 ? (rows + kWarps - 1) / kWarps : 148 * 8); }

// Sums over the splits of row b of its N values, which lie in shared memory or were Written by the kernel before.  A row of many
// splits is added up by a warp, whose lanes all call this.
constexpr int kSplitsPerThread = 8;
template <int N, typename Part>
__device__ __forceinline__ void row_sums(const Part& part, long long b, int splits, double (&row)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < N; ++i) row[i] = 0.;
  if (splits <= kSplitsPerThread) {
    for (int s = 0; s < splits; ++s)
      for (int i = 0; i < N; ++i) row[i] += part[(b * splits + s) * N + i];
    return;
  }
  for (int s = lane; s < splits; s += 32)
    for (int i = 0; i < N; ++i) row[i] += part[(b * splits + s) * N + i];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) row[i] += __shfl_xor_sync(~0u, row[i], o);
}
// The rows this thread works on in a finishing block: each thread its own, or each warp its own.
__device__ __forceinline__ long long first_row(int splits) { return splits <= kSplitsPerThread ? threadIdx.x : threadIdx.x >> 5; }
__device__ __forceinline__ int row_step(int splits) { return splits <= kSplitsPerThread ? blockDim.x : blockDim.x >> 5; }
__device__ __forceinline__ bool speaks(int splits) { return splits <= kSplitsPerThread || (threadIdx.x & 31) == 0; }

// ---- clipped policy loss -------------------------------------------------------------------------------------------
struct PolicyArgs {
  const float *logprob, *old, *ref, *advantage;
  const uint8_t* mask;
  long long lp_stride, old_stride, ref_stride, adv_stride, mask_stride;
  long long batch;
  int seq, per_token, splits, part;   // part: tokens of one of the splits of a row
  double log_high, log_low;   // ln(1 + clip_high), ln(1 - clip_low): the borders of ln r
  float log_high_f, log_low_f, above, below, kl_coef;   // the borders rounded to fp32; the clamp's ends less one
};

// (exp(d) - 1 - d) / d^2 for |d| <= 1: the Taylor series 1/2! + d (1/3! + d (1/4! + ...)) to the term d^12 of the exponential;
// what it leaves out is below 2/13! < 2^-31 of the result.  Nearly all tokens of a policy near the one that sampled, and near
// its reference, lie in this range, so that a warp seldom takes the other way as well.
__device__ __forceinline__ float exp_tail(float d) {
  constexpr float kInverseFactorial[] = {1.f / 2, 1.f / 6, 1.f / 24, 1.f / 120, 1.f / 720, 1.f / 5040, 1.f / 40320, 1.f / 362880,
                                         1.f / 3628800, 1.f / 39916800, 1.f / 479001600};
  float r = kInverseFactorial[10];
#pragma unroll
  for (int k = 9; k >= 0; --k) r = fmaf(r, d, kInverseFactorial[k]);
  return r;
}
// r = exp(d) and less = r - 1, both to a few roundings of their own size.
__device__ __forceinline__ void ratio(float d, float& r, float& less) {
  if (fabsf(d) <= 1.f) {
    less = fmaf(d * d, exp_tail(d), d);
    r = 1.f + less;
  } else {
    r = expf(d);
    less = r - 1.f;
  }
}
// k = exp(d) - 1 - d and slope = exp(d) - 1.
__device__ __forceinline__ void divergence(float d, float& k, float& slope) {
  if (fabsf(d) <= 1.f) {
    const float tail = exp_tail(d);
    k = d * d * tail;
    slope = fmaf(d * d, tail, d);
  } else {
    slope = expm1f(d);
    k = d > 60.f ? slope : slope - d;   // 1 + d is below the last bit; an infinite d must not meet itself
  }
}

// Tokens begin, begin + step, ... below end of row b, kUnroll of them loaded at a time; full rounds need no bounds checks.
template <bool REF, bool MASK>
__device__ __forceinline__ void policy_tokens(const PolicyArgs& a, long long b, int begin, int end, int step,
                                              float* __restrict__ unit_grad, Sums<2, 2>& sum) {
  const float* lp_row = a.logprob + b * a.lp_stride;
  const float* old_row = a.old + b * a.old_stride;
  const float* ref_row = REF ? a.ref + b * a.ref_stride : nullptr;
  const uint8_t* mask_row = MASK ? a.mask + b * a.mask_stride : nullptr;
  const float* adv_row = a.advantage + b * a.adv_stride;
  const float one_adv = !a.per_token && begin < end ? adv_row[0] : 0.f;
  float* unit_row = unit_grad != nullptr ? unit_grad + b * a.seq : nullptr;
  const auto round = [&](int t0, auto full) {
    constexpr bool FULL = decltype(full)::value;
    float lp[kUnroll], old[kUnroll], adv[kUnroll], ref[kUnroll];
    bool kept[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int t = FULL || t0 + j * step < end ? t0 + j * step : t0;   // a token of the row in any case
      lp[j] = lp_row[t];
      old[j] = old_row[t];
      adv[j] = a.per_token ? adv_row[t] : one_adv;
      if (REF) ref[j] = ref_row[t];
      kept[j] = (FULL || t0 + j * step < end) && (!MASK || mask_row[t] != 0);
    }
    float loss = 0.f, ks = 0.f;
    double level = 0.;
    int cuts = 0, keeps = 0;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      // fp32 rounds monotonously, so the rounded difference decides the border unless it lies on it
      const float d = lp[j] - old[j];
      bool cut = (adv[j] > 0.f && d > a.log_high_f) || (adv[j] < 0.f && d < a.log_low_f);
      if (d == a.log_high_f || d == a.log_low_f) {
        const double exact = (double)lp[j] - (double)old[j];
        cut = (adv[j] > 0.f && exact > a.log_high) || (adv[j] < 0.f && exact < a.log_low);
      }
      float r, less;
      ratio(d, r, less);
      // -r A as -A, added in 64 bits, and -(r - 1) A, which is small near the policy that sampled: advantages of both signs
      // cancel in the mean, the rounding of products of order one would not.  The product with an advantage of zero is zero
      // however large the ratio; a NaN stays one.
      const bool nothing = adv[j] == 0.f && !isnan(d);
      const float rest = nothing ? 0.f : -(cut ? (adv[j] > 0.f ? a.above : a.below) : less) * adv[j];
      float g = cut || nothing ? 0.f : -r * adv[j];
      if (REF) {
        float k, slope;
        divergence(ref[j] - lp[j], k, slope);
        if (a.kl_coef != 0.f) g -= a.kl_coef * slope;
        ks += kept[j] ? k : 0.f;
      }
      loss += kept[j] ? rest : 0.f;
      level -= kept[j] ? (double)adv[j] : 0.;
      cuts += kept[j] && cut;
      keeps += kept[j];
      if (unit_row != nullptr && (FULL || t0 + j * step < end)) unit_row[t0 + j * step] = kept[j] ? g : 0.f;
    }
    // the small parts of four tokens in fp32, then in 64 bits
    sum.v[0] += level + (double)loss;
    if (REF) sum.v[1] += ks;
    sum.n[0] += cuts;
    sum.n[1] += keeps;
  };
  int t0 = begin;
  for (; t0 + (kUnroll - 1) * step < end; t0 += kUnroll * step) round(t0, Full{});
  if (t0 < end) round(t0, Ragged{});
}

// What a row adds to the mean: its sums (loss, k, cut) times its own weight, 1 or 1 / its length, and its share of the
// divisor, its length or 1.  The divisor is known last; it goes behind the rows' weights, and the backward multiplies both.
__device__ __forceinline__ double add_row(const double (&row)[4], int reduction, double (&sum)[4]) {
  if (!(row[3] > 0.)) return 0.;
  const double w = reduction == MOLT_REDUCE_TOKEN ? 1. : 1. / row[3];
  for (int i = 0; i < 3; ++i) sum[i] += w * row[i];
  sum[3] += w * row[3];
  return w;
}

__device__ __forceinline__ void policy_result(double (&sum)[4], double kl_coef, float* __restrict__ scale,
                                              float* __restrict__ loss, float* __restrict__ stats) {
  block_sum(sum);
  if (threadIdx.x == 0) {
    const double one = sum[3] > 0. ? 1. / sum[3] : 0.;
    loss[0] = (float)((kl_coef != 0. ? sum[0] + kl_coef * sum[1] : sum[0]) * one);
    stats[0] = (float)(sum[1] * one);
    stats[1] = (float)(sum[2] * one);
    if (scale != nullptr) scale[0] = (float)one;
  }
}

// Rows, their weights and the result, by one block.
template <typename Part>
__device__ __forceinline__ void policy_finish(const Part& part, long long batch, int splits, int reduction, double kl_coef,
                                              float* __restrict__ row_weight, float* __restrict__ loss,
                                              float* __restrict__ stats) {
  double sum[4] = {0., 0., 0., 0.};
  for (long long b = first_row(splits); b < batch; b += row_step(splits)) {
    double row[4];
    row_sums(part, b, splits, row);
    if (speaks(splits)) {
      const double w = add_row(row, reduction, sum);
      if (row_weight != nullptr) row_weight[b] = (float)w;
    }
  }
  policy_result(sum, kl_coef, row_weight != nullptr ? row_weight + batch : nullptr, loss, stats);
}

template <bool REF, bool MASK>
__global__ void __launch_bounds__(kThreads, 5) policy_kernel(PolicyArgs a, float* __restrict__ unit_grad,
                                                             double* __restrict__ part) {
  let_next_begin();
  const long long b = blockIdx.x;
  const int begin = blockIdx.y * a.part;
  __shared__ double of_warp[4 * 32];
  Sums<2, 2> sum;   // loss, k; cut, kept
  policy_tokens<REF, MASK>(a, b, begin + threadIdx.x, min(a.seq, begin + a.part), kThreads, unit_grad, sum);
  sum.join_warp();
  if ((threadIdx.x & 31) == 0) sum.store(of_warp + (threadIdx.x >> 5), 32);
  const double mine = join_block(of_warp, 4);
  const int value = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0 && value < 4) part[(b * a.splits + blockIdx.y) * 4 + value] = mine;
}

__global__ void __launch_bounds__(kFinish) policy_finish_kernel(const Written part, long long batch, int splits,
                                                             int reduction, double kl_coef, float* __restrict__ row_weight,
                                                             float* __restrict__ loss, float* __restrict__ stats) {
  wait_for_previous();
  policy_finish(part, batch, splits, reduction, kl_coef, row_weight, loss, stats);
}

// A warp per row: what the block's rows add to the mean goes to part[block].
template <bool REF, bool MASK>
__global__ void __launch_bounds__(kThreads, 4) policy_rows_kernel(PolicyArgs a, int reduction, float* __restrict__ unit_grad,
                                                                  float* __restrict__ row_weight, double* __restrict__ part) {
  let_next_begin();
  __shared__ double of_warp[4 * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum[4] = {0., 0., 0., 0.};
  for (long long b = (long long)blockIdx.x * kWarps + warp; b < a.batch; b += (long long)gridDim.x * kWarps) {
    Sums<2, 2> one;
    policy_tokens<REF, MASK>(a, b, lane, a.seq, 32, unit_grad, one);
    one.join_warp();
    const double row[4] = {one.v[0], one.v[1], (double)one.n[0], (double)one.n[1]};
    const double w = add_row(row, reduction, sum);
    if (lane == 0 && row_weight != nullptr) row_weight[b] = (float)w;
  }
  if (lane == 0)
    for (int i = 0; i < 4; ++i) of_warp[i * 32 + warp] = sum[i];
  const double mine = join_block(of_warp, 4);
  if (lane == 0 && warp < 4) part[blockIdx.x * 4 + warp] = mine;
}

__global__ void __launch_bounds__(kFinish) policy_rows_finish_kernel(const Written part, int blocks, double kl_coef,
                                                                     float* __restrict__ scale, float* __restrict__ loss,
                                                                     float* __restrict__ stats) {
  wait_for_previous();
  double sum[4] = {0., 0., 0., 0.};
  for (int k = threadIdx.x; k < blocks; k += blockDim.x)
    for (int i = 0; i < 4; ++i) sum[i] += part[k * 4 + i];
  policy_result(sum, kl_coef, scale, loss, stats);
}

// The whole forward in one block: a warp takes one of the splits of a row.
template <bool REF, bool MASK>
__global__ void __launch_bounds__(kOneBlock) policy_one_block_kernel(PolicyArgs a, int reduction, double kl_coef,
                                                                     float* __restrict__ unit_grad,
                                                                     float* __restrict__ row_weight, float* __restrict__ loss,
                                                                     float* __restrict__ stats) {
  __shared__ double part[kOneBlockRows * 4];
  const int lane = threadIdx.x & 31, units = (int)a.batch * a.splits;
  for (int u = threadIdx.x >> 5; u < units; u += kOneBlock / 32) {
    const int b = u / a.splits, s = u - b * a.splits;
    Sums<2, 2> sum;
    policy_tokens<REF, MASK>(a, b, s * a.part + lane, min(a.seq, (s + 1) * a.part), 32, unit_grad, sum);
    sum.join_warp();
    if (lane == 0) sum.store(part + u * 4, 1);
  }
  __syncthreads();
  policy_finish(part, a.batch, a.splits, reduction, kl_coef, row_weight, loss, stats);
}

// Backward passes.  A block is one round of one row; where rows are short (SHORT) it is one round of all tokens, numbered
// through, and every token looks its row up (65536 x 16 tokens with a block per row: 37 us).
constexpr int kShort = kRound / 2;

struct Place {
  long long row, token, flat;
  bool valid;
};
template <bool SHORT>
__device__ __forceinline__ Place place(long long rows, int seq, int j) {
  Place p;
  if (SHORT) {
    p.flat = (long long)blockIdx.x * kRound + j * kThreads + threadIdx.x;
    p.valid = p.flat < rows * seq;
    // 32-bit division where it is enough
    p.row = rows * seq <= 0xffffffffLL ? (long long)((unsigned)p.flat / (unsigned)seq) : p.flat / seq;
    p.token = p.flat - p.row * seq;
  } else {
    p.row = blockIdx.x;
    p.token = (long long)blockIdx.y * kRound + j * kThreads + threadIdx.x;
    p.flat = p.row * seq + p.token;
    p.valid = p.token < seq;
  }
  return p;
}
bool short_rows(int64_t rows, int64_t seq) { return seq <= kShort && (rows * seq + kRound - 1) / kRound < (1LL << 31); }
dim3 backward_grid(int64_t rows, int64_t seq) {
  return short_rows(rows, seq) ? dim3((unsigned)((rows * seq + kRound - 1) / kRound))
                               : dim3((unsigned)rows, (unsigned)((seq + kRound - 1) / kRound));
}

template <bool SHORT>
__global__ void __launch_bounds__(kThreads) policy_backward_kernel(const float* __restrict__ unit_grad,
                                                                   const float* __restrict__ row_weight,
                                                                   const float* __restrict__ grad_loss,
                                                                   float* __restrict__ grad_logprob, long long batch, int seq) {
  float u[kUnroll], w[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {   // all loads before the first store
    const Place p = place<SHORT>(batch, seq, j);
    u[j] = p.valid ? unit_grad[p.flat] : 0.f;
    w[j] = SHORT ? (p.valid ? row_weight[p.row] : 0.f) : row_weight[blockIdx.x];
  }
  const float g = row_weight[batch] * grad_loss[0];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const Place p = place<SHORT>(batch, seq, j);
    if (p.valid) grad_logprob[p.flat] = u[j] == 0.f ? 0.f : u[j] * (w[j] * g);
  }
}

// ---- preference pairs ----------------------------------------------------------------------------------------------
struct PreferenceArgs {
  const float *logprob, *ref;
  const uint8_t* mask;
  long long lp_stride, ref_stride, mask_stride;
  long long pairs;
  int seq, ref_per_token, splits, part, kind, average;   // part: tokens of one of the splits of a row
  double beta, smoothing;
};

template <bool REF, bool MASK>
__device__ __forceinline__ void preference_tokens(const PreferenceArgs& a, long long i, int begin, int end, int step,
                                                  Sums<1, 1>& sum) {
  const float* lp_row = a.logprob + i * a.lp_stride;
  const float* ref_row = REF ? a.ref + i * a.ref_stride : nullptr;
  const uint8_t* mask_row = MASK ? a.mask + i * a.mask_stride : nullptr;
  const auto round = [&](int t0, auto full) {
    constexpr bool FULL = decltype(full)::value;
    float lp[kUnroll], ref[kUnroll];
    bool kept[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int t = FULL || t0 + j * step < end ? t0 + j * step : t0;   // a token of the row in any case
      lp[j] = lp_row[t];
      if (REF) ref[j] = ref_row[t];
      kept[j] = (FULL || t0 + j * step < end) && (!MASK || mask_row[t] != 0);
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      // in 64 bits from the start: the differences of a sequence cancel, their rounding would not
      if (kept[j]) sum.v[0] += REF ? (double)lp[j] - (double)ref[j] : (double)lp[j];
      sum.n[0] += kept[j];
    }
  };
  int t0 = begin;
  for (; t0 + (kUnroll - 1) * step < end; t0 += kUnroll * step) round(t0, Full{});
  if (t0 < end) round(t0, Ragged{});
}

template <typename Part>
__device__ __forceinline__ void preference_finish(const PreferenceArgs& a, const Part& part, float* __restrict__ seq_grad,
                                                  float* __restrict__ rewards, float* __restrict__ loss_out) {
  double total[1] = {0.};
  for (long long p = first_row(a.splits); p < a.pairs; p += row_step(a.splits)) {
    double s[2], scale[2];
    for (int side = 0; side < 2; ++side) {
      const long long i = p + side * a.pairs;
      double row[2];
      row_sums(part, i, a.splits, row);
      const double sum = row[0], kept = row[1];
      scale[side] = a.average ? (kept > 0. ? 1. / kept : 0.) : 1.;
      s[side] = a.average ? (kept > 0. ? sum / kept : 0.) : sum;
      if (a.ref != nullptr && !a.ref_per_token) s[side] -= (double)a.ref[i * a.ref_stride];
      if (speaks(a.splits)) rewards[i] = (float)(a.beta * s[side]);
    }
    if (!speaks(a.splits)) continue;
    const double h = s[0] - s[1];
    double loss, slope;
    if (a.kind == MOLT_PREFERENCE_SIGMOID) {
      const double z = a.beta * h, e = exp(-fabs(z)), soft = log1p(e);   // -ln sig(z) = soft + max(-z, 0)
      loss = soft;                                                       // an infinite z must not meet a factor of zero
      if (a.smoothing != 1.) loss += (1. - a.smoothing) * fmax(-z, 0.);
      if (a.smoothing != 0.) loss += a.smoothing * fmax(z, 0.);
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

template <bool REF, bool MASK>
__global__ void __launch_bounds__(kThreads, 8) preference_kernel(PreferenceArgs a, double* __restrict__ part) {
  let_next_begin();
  const long long i = blockIdx.x;
  const int begin = blockIdx.y * a.part;
  __shared__ double of_warp[2 * 32];
  Sums<1, 1> sum;   // difference to the reference; kept
  preference_tokens<REF, MASK>(a, i, begin + threadIdx.x, min(a.seq, begin + a.part), kThreads, sum);
  sum.join_warp();
  if ((threadIdx.x & 31) == 0) sum.store(of_warp + (threadIdx.x >> 5), 32);
  const double mine = join_block(of_warp, 2);
  const int value = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0 && value < 2) part[(i * a.splits + blockIdx.y) * 2 + value] = mine;
}

// A warp per row.
template <bool REF, bool MASK>
__global__ void __launch_bounds__(kThreads, 8) preference_rows_kernel(PreferenceArgs a, double* __restrict__ part) {
  let_next_begin();
  const int lane = threadIdx.x & 31;
  for (long long i = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); i < 2 * a.pairs; i += (long long)gridDim.x * kWarps) {
    Sums<1, 1> sum;
    preference_tokens<REF, MASK>(a, i, lane, a.seq, 32, sum);
    sum.join_warp();
    if (lane == 0) sum.store(part + i * 2, 1);
  }
}

__global__ void __launch_bounds__(kFinish) preference_finish_kernel(PreferenceArgs a, const Written part,
                                                                 float* __restrict__ seq_grad, float* __restrict__ rewards,
                                                                 float* __restrict__ loss) {
  wait_for_previous();
  preference_finish(a, part, seq_grad, rewards, loss);
}

template <bool REF, bool MASK>
__global__ void __launch_bounds__(kOneBlock) preference_one_block_kernel(PreferenceArgs a, float* __restrict__ seq_grad,
                                                                         float* __restrict__ rewards, float* __restrict__ loss) {
  __shared__ double part[kOneBlockRows * 2];
  const int lane = threadIdx.x & 31, units = (int)(2 * a.pairs) * a.splits;
  for (int u = threadIdx.x >> 5; u < units; u += kOneBlock / 32) {
    const int i = u / a.splits, s = u - i * a.splits;
    Sums<1, 1> sum;
    preference_tokens<REF, MASK>(a, i, s * a.part + lane, min(a.seq, (s + 1) * a.part), 32, sum);
    sum.join_warp();
    if (lane == 0) sum.store(part + u * 2, 1);
  }
  __syncthreads();
  preference_finish(a, part, seq_grad, rewards, loss);
}

template <bool SHORT>
__global__ void __launch_bounds__(kThreads) preference_backward_kernel(const uint8_t* __restrict__ mask, long long mask_stride,
                                                                       const float* __restrict__ seq_grad,
                                                                       const float* __restrict__ grad_loss,
                                                                       float* __restrict__ grad_logprob, long long rows, int seq) {
  const float one = SHORT ? 0.f : seq_grad[blockIdx.x], g = grad_loss[0];
  float w[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {   // all loads before the first store
    const Place p = place<SHORT>(rows, seq, j);
    const float of_row = SHORT ? (p.valid ? seq_grad[p.row] : 0.f) : one;
    w[j] = p.valid && (mask == nullptr || mask[p.row * mask_stride + p.token] != 0) ? of_row : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const Place p = place<SHORT>(rows, seq, j);
    if (p.valid) grad_logprob[p.flat] = w[j] == 0.f ? 0.f : w[j] * g;
  }
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
  return (warp_rows(batch, seq) ? (size_t)warp_row_blocks(batch) : (size_t)batch * splits_for(batch, seq)) * 4 * sizeof(double);
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
  a.batch = batch; a.seq = (int)seq; a.per_token = advantage_per_token != 0;
  a.splits = splits_for(batch, seq); a.part = part_tokens(batch, seq);
  a.log_high = log1p(clip_high); a.log_low = log1p(-clip_low);
  a.log_high_f = (float)a.log_high; a.log_low_f = (float)a.log_low;
  a.above = (float)clip_high; a.below = (float)-clip_low; a.kl_coef = (float)kl_coef;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (needed == 0) {
    a.splits = one_block_splits(batch);
    a.part = ((int)seq + a.splits - 1) / a.splits;
    const auto kernel = ref_logprob != nullptr ? (mask != nullptr ? policy_one_block_kernel<true, true> : policy_one_block_kernel<true, false>)
                                               : (mask != nullptr ? policy_one_block_kernel<false, true> : policy_one_block_kernel<false, false>);
    kernel<<<1, kOneBlock, 0, s>>>(a, reduction, kl_coef, unit_grad, row_weight, loss, stats);
    return launch_status("policy_one_block_kernel");
  }
  auto* part = reinterpret_cast<double*>(workspace);
  if (warp_rows(batch, seq)) {
    const int blocks = warp_row_blocks(batch);
    const auto kernel = ref_logprob != nullptr ? (mask != nullptr ? policy_rows_kernel<true, true> : policy_rows_kernel<true, false>)
                                               : (mask != nullptr ? policy_rows_kernel<false, true> : policy_rows_kernel<false, false>);
    kernel<<<blocks, kThreads, 0, s>>>(a, reduction, unit_grad, row_weight, part);
    if (int rc = launch_status("policy_rows_kernel")) return rc;
    launch_behind(policy_rows_finish_kernel, 1, kFinish, s, part, blocks, kl_coef,
                  row_weight != nullptr ? row_weight + batch : nullptr, loss, stats);
    return launch_status("policy_rows_finish_kernel");
  }
  const auto kernel = ref_logprob != nullptr ? (mask != nullptr ? policy_kernel<true, true> : policy_kernel<true, false>)
                                             : (mask != nullptr ? policy_kernel<false, true> : policy_kernel<false, false>);
  kernel<<<dim3((unsigned)batch, a.splits), kThreads, 0, s>>>(a, unit_grad, part);
  if (int rc = launch_status("policy_kernel")) return rc;
  launch_behind(policy_finish_kernel, 1, kFinish, s, part, (long long)batch, a.splits, reduction, kl_coef, row_weight, loss, stats);
  return launch_status("policy_finish_kernel");
}

extern "C" int molt_policy_loss_bwd(const float* unit_grad, const float* row_weight, const float* grad_loss, float* grad_logprob,
                                    int64_t batch, int64_t seq, uintptr_t stream) {
  const char* who = "molt_policy_loss_bwd";
  if (int rc = check_sizes(who, batch, seq)) return rc;
  if (batch == 0 || seq == 0) return MOLT_OK;
  MOLT_REQUIRE(unit_grad && row_weight && grad_loss && grad_logprob, MOLT_E_VALUE, "%s: NULL tensor pointer", who);
  const auto kernel = short_rows(batch, seq) ? policy_backward_kernel<true> : policy_backward_kernel<false>;
  kernel<<<backward_grid(batch, seq), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(unit_grad, row_weight, grad_loss,
                                                                                            grad_logprob, batch, (int)seq);
  return launch_status("policy_backward_kernel");
}

extern "C" size_t molt_preference_loss_workspace_bytes(int64_t pairs, int64_t seq) {
  if (pairs <= 0 || seq < 0 || one_block(2 * pairs, seq)) return 0;
  return (size_t)pairs * 2 * (warp_rows(2 * pairs, seq) ? 1 : splits_for(pairs * 2, seq)) * 2 * sizeof(double);
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
  a.pairs = pairs; a.seq = (int)seq; a.ref_per_token = ref_per_token != 0;
  a.splits = splits_for(2 * pairs, seq); a.part = part_tokens(2 * pairs, seq);
  const bool tokens = ref_logprob != nullptr && ref_per_token;   // the reference is subtracted token by token
  a.kind = kind; a.average = average != 0; a.beta = beta; a.smoothing = smoothing;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (needed == 0) {
    a.splits = one_block_splits(2 * pairs);
    a.part = ((int)seq + a.splits - 1) / a.splits;
    const auto kernel = tokens ? (mask != nullptr ? preference_one_block_kernel<true, true> : preference_one_block_kernel<true, false>)
                               : (mask != nullptr ? preference_one_block_kernel<false, true> : preference_one_block_kernel<false, false>);
    kernel<<<1, kOneBlock, 0, s>>>(a, seq_grad, rewards, loss);
    return launch_status("preference_one_block_kernel");
  }
  auto* part = reinterpret_cast<double*>(workspace);
  if (warp_rows(2 * pairs, seq)) {
    a.splits = 1;
    const auto kernel = tokens ? (mask != nullptr ? preference_rows_kernel<true, true> : preference_rows_kernel<true, false>)
                               : (mask != nullptr ? preference_rows_kernel<false, true> : preference_rows_kernel<false, false>);
    kernel<<<warp_row_blocks(2 * pairs), kThreads, 0, s>>>(a, part);
    if (int rc = launch_status("preference_rows_kernel")) return rc;
    launch_behind(preference_finish_kernel, 1, kFinish, s, a, part, seq_grad, rewards, loss);
    return launch_status("preference_finish_kernel");
  }
  const auto kernel = tokens ? (mask != nullptr ? preference_kernel<true, true> : preference_kernel<true, false>)
                             : (mask != nullptr ? preference_kernel<false, true> : preference_kernel<false, false>);
  kernel<<<dim3((unsigned)(2 * pairs), a.splits), kThreads, 0, s>>>(a, part);
  if (int rc = launch_status("preference_kernel")) return rc;
  launch_behind(preference_finish_kernel, 1, kFinish, s, a, part, seq_grad, rewards, loss);
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
  const auto kernel = short_rows(2 * pairs, seq) ? preference_backward_kernel<true> : preference_backward_kernel<false>;
  kernel<<<backward_grid(2 * pairs, seq), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      mask, mask_stride, seq_grad, grad_loss, grad_logprob, 2 * pairs, (int)seq);
  return launch_status("preference_backward_kernel");
}

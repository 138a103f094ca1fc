// A router's load: slots per expert, and the load-balance loss with its
// gradient.
//
// n rows count (those not marked as padding), c_e of their k slots chose expert
// e, f_e = E c_e / (n k) (1 for even load).  With p_t the row's probabilities
// (softmax of its logits, or its sigmoids over their sum),
//
//   loss = sum_e f_e (1/n) sum_t p_te = (1/n) sum_t r_t,   r_t = sum_e f_e p_te,
//
// so that no expert's mean probability is needed: a row's part of the loss and
// its gradient (g the loss's own gradient, the counts constants),
//
//   softmax:  dloss/dl_te = g/n p_te (f_e - r_t)
//   sigmoid:  dloss/dl_te = g/n p_te (1 - s_te) (f_e - r_t),  s_te the sigmoid,
//
// come from the counts and the row alone.  The forward reads the logits once
// and the backward once more (keeping the probabilities would write and read as
// much).  A row whose logits leave nothing (all -inf, sigmoids that sum to 0)
// has p = 0.  Counts are whole numbers, so their atomics give one result in any
// order; the rows' parts are summed in 64 bits in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/vllm_mi355x.h"
#include "common.h"

namespace balance {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kMaxParts = 64;    // workgroups that count
constexpr int kMaxGroups = 1024; // workgroups that take rows

__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += vq::xor_lanes<32>(v, lane);
  v += vq::xor_lanes<16>(v, lane);
  v += vq::xor_lanes<8>(v, lane);
  v += vq::xor_lanes<4>(v, lane);
  v += vq::xor_lanes<2>(v, lane);
  v += vq::xor_lanes<1>(v, lane);
  return v;
}

// hist[part][E + 1]: the part's slots by expert, and its rows.
__global__ __launch_bounds__(kThreads) void count_kernel(const int32_t* ids, const uint8_t* padding, int64_t rows, int top_k,
                                                         int experts, int32_t* hist) {
  extern __shared__ int count[];
  for (int e = threadIdx.x; e <= experts; e += kThreads) count[e] = 0;
  __syncthreads();
  int mine = 0;
  for (int64_t t = int64_t(blockIdx.x) * kThreads + threadIdx.x; t < rows; t += int64_t(gridDim.x) * kThreads) {
    if (padding && padding[t]) continue;
    ++mine;
    for (int k = 0; k < top_k; ++k) {
      const int id = ids[t * top_k + k];
      if (id >= 0 && id < experts) atomicAdd(&count[id], 1);
    }
  }
  if (mine) atomicAdd(&count[experts], mine);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kThreads) hist[int64_t(blockIdx.x) * (experts + 1) + e] = count[e];
}

// counts[e] (+)= the parts' sums; stats (may be null): f_e, then 1/n (0 for no rows).
__global__ __launch_bounds__(kThreads) void totals_kernel(const int32_t* hist, int parts, int experts, int top_k, bool add,
                                                          int64_t* counts, float* stats) {
  int64_t n = 0;
  for (int p = 0; p < parts; ++p) n += hist[int64_t(p) * (experts + 1) + experts];
  for (int e = threadIdx.x; e < experts; e += kThreads) {
    int64_t c = 0;
    for (int p = 0; p < parts; ++p) c += hist[int64_t(p) * (experts + 1) + e];
    counts[e] = add ? counts[e] + c : c;
    if (stats) stats[e] = n ? float(double(c) * experts / (double(n) * top_k)) : 0.0f;
  }
  if (stats && threadIdx.x == 0) stats[experts] = n ? float(1.0 / double(n)) : 0.0f;
}

// The row's probabilities p and, for the gradient, their slopes d (lane holds
// experts lane + 64 i), and r = sum f p.
template <int kPer, bool kSigmoid>
__device__ __forceinline__ float row_terms(const void* logits, int dtype, int64_t at, const float* f, int experts, int lane,
                                           float (&d)[kPer]) {
  float l[kPer], z[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 64 * i;
    l[i] = e < experts ? vq::load_act(logits, dtype, at + e) : -__builtin_inff();
  }
  float m = 0;
  if constexpr (!kSigmoid) {
    m = l[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) m = fmaxf(m, l[i]);
    m = vq::wave_max(m, lane);
    if (m == -__builtin_inff()) m = 0;
  }
  float sum = 0, dot = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + 64 * i;
    if constexpr (kSigmoid) {
      const float t = expf(-fabsf(l[i]));
      const float small = t / (1 + t), large = 1 / (1 + t);
      z[i] = l[i] >= 0 ? large : small;
      d[i] = l[i] >= 0 ? small : large;
    } else {
      z[i] = expf(l[i] - m);
      d[i] = 1;
    }
    if (e < experts) {
      sum += z[i];
      dot += f[e] * z[i];
    }
  }
  sum = wave_sum(sum, lane);
  dot = wave_sum(dot, lane);
  const float inv = sum == 0 ? 0.0f : 1 / sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) d[i] *= z[i] * inv;
  return dot * inv;
}

// partial[workgroup] = the sum of its rows' r, one row a wavefront.
template <int kPer, bool kSigmoid>
__global__ __launch_bounds__(kThreads) void loss_kernel(const void* logits, int dtype, int64_t stride, const uint8_t* padding,
                                                        int64_t rows, int experts, const float* stats, double* partial) {
  __shared__ double part[kWaves];
  const int lane = threadIdx.x & 63, wave = vq::uniform(int(threadIdx.x) >> 6);
  double sum = 0;
  float d[kPer];
  for (int64_t t = int64_t(blockIdx.x) * kWaves + wave; t < rows; t += int64_t(gridDim.x) * kWaves) {
    if (padding && padding[t]) continue;
    sum += row_terms<kPer, kSigmoid>(logits, dtype, t * stride, stats, experts, lane, d);
  }
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0;
    for (int w = 0; w < kWaves; ++w) all += part[w];
    partial[blockIdx.x] = all;
  }
}

__global__ __launch_bounds__(64) void finish_kernel(const double* partial, int groups, const float* inv_n, float* loss) {
  __shared__ double part[64];
  double sum = 0;
  for (int i = threadIdx.x; i < groups; i += 64) sum += partial[i];
  part[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0;
    for (int i = 0; i < 64; ++i) all += part[i];
    loss[0] = float(all * double(inv_n[0]));
  }
}

template <int kPer, bool kSigmoid>
__global__ __launch_bounds__(kThreads) void grad_kernel(const void* logits, int dtype, int64_t stride, const uint8_t* padding,
                                                        int64_t rows, int experts, const float* stats, const float* upstream,
                                                        void* grad) {
  const int lane = threadIdx.x & 63, wave = vq::uniform(int(threadIdx.x) >> 6);
  const float scale = upstream[0] * stats[experts];
  float d[kPer];
  for (int64_t t = int64_t(blockIdx.x) * kWaves + wave; t < rows; t += int64_t(gridDim.x) * kWaves) {
    const bool counted = !(padding && padding[t]);
    float r = 0;
    if (counted) r = row_terms<kPer, kSigmoid>(logits, dtype, t * stride, stats, experts, lane, d);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 64 * i;
      if (e < experts) vq::store_act(grad, dtype, t * experts + e, counted ? scale * d[i] * (stats[e] - r) : 0.0f);
    }
  }
}

template <typename F>
int by_width(int64_t experts, bool sigmoid, const F& launch) {
  const auto pick = [&](auto per) {
    if (sigmoid) launch(per, std::true_type{});
    else launch(per, std::false_type{});
  };
  if (experts <= 64) pick(std::integral_constant<int, 1>{});
  else if (experts <= 128) pick(std::integral_constant<int, 2>{});
  else if (experts <= 256) pick(std::integral_constant<int, 4>{});
  else if (experts <= 512) pick(std::integral_constant<int, 8>{});
  else pick(std::integral_constant<int, 16>{});
  return vq::check_launch("moe balance");
}

int64_t parts_of(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(kMaxParts, (rows + kThreads - 1) / kThreads)); }
int64_t groups_of(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(kMaxGroups, (rows + kWaves - 1) / kWaves)); }

int check_sizes(int64_t rows, int64_t experts, int64_t top_k) {
  if (rows < 0 || rows > INT_MAX) return vq::fail("moe balance: rows out of range");
  if (experts <= 0 || experts > kMaxExperts) return vq::fail("moe balance: between 1 and 1024 experts");
  if (top_k <= 0 || top_k > INT_MAX || rows * top_k > INT_MAX) return vq::fail("moe balance: top_k out of range");
  return vq::kOk;
}

int launch_counts(const int32_t* ids, const uint8_t* padding, int64_t rows, int64_t top_k, int64_t experts, bool add,
                  int64_t* counts, float* stats, int32_t* hist, hipStream_t s) {
  const int parts = int(parts_of(rows));
  hipLaunchKernelGGL(count_kernel, dim3(unsigned(parts)), dim3(kThreads), size_t(experts + 1) * sizeof(int), s, ids, padding, rows,
                     int(top_k), int(experts), hist);
  if (int rc = vq::check_launch("moe counts")) return rc;
  hipLaunchKernelGGL(totals_kernel, dim3(1), dim3(kThreads), 0, s, hist, parts, int(experts), int(top_k), add, counts, stats);
  return vq::check_launch("moe counts");
}

int check_logits(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, int scoring) {
  if (dtype != vq::kBF16 && dtype != vq::kFP16 && dtype != vq::kFP32) return vq::fail("moe balance: logits must be BF16, FP16 or FP32");
  if (scoring != 0 && scoring != 1) return vq::fail("moe balance: scoring must be softmax (0) or sigmoid (1)");
  if (stride < 0 || (rows > 1 && stride < experts) || stride > (int64_t(1) << 31)) return vq::fail("moe balance: row stride out of range");
  if (rows > 0 && !logits) return vq::fail("moe balance: null pointer");
  return vq::kOk;
}

bool aligned8(const void* p) { return reinterpret_cast<uintptr_t>(p) % 8 == 0; }

}  // namespace
}  // namespace balance

extern "C" int64_t moe_balance_workspace_size(int64_t rows, int64_t experts) {
  using namespace balance;
  if (check_sizes(rows, experts, 1)) return -1;
  return kMaxGroups * int64_t(sizeof(double)) + parts_of(rows) * (experts + 1) * int64_t(sizeof(int32_t));
}

extern "C" int moe_expert_counts(const int32_t* topk_ids, const uint8_t* is_padding, int64_t rows, int64_t top_k, int64_t experts,
                                 int add, int64_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, top_k)) return rc;
  if (!counts || !workspace || (rows > 0 && !topk_ids)) return vq::fail("moe balance: null pointer");
  if (workspace_bytes < moe_balance_workspace_size(rows, experts) || !aligned8(workspace)) return vq::fail("moe balance: workspace too small or misaligned");
  int32_t* hist = reinterpret_cast<int32_t*>(static_cast<double*>(workspace) + kMaxGroups);
  return launch_counts(topk_ids, is_padding, rows, top_k, experts, add != 0, counts, nullptr, hist, static_cast<hipStream_t>(stream));
}

extern "C" int moe_balance_loss(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const int32_t* topk_ids,
                                int64_t top_k, const uint8_t* is_padding, int scoring, float* loss, int64_t* counts, float* stats,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, top_k)) return rc;
  if (int rc = check_logits(logits, dtype, rows, experts, stride, scoring)) return rc;
  if (!loss || !counts || !stats || !workspace || (rows > 0 && !topk_ids)) return vq::fail("moe balance: null pointer");
  if (workspace_bytes < moe_balance_workspace_size(rows, experts) || !aligned8(workspace)) return vq::fail("moe balance: workspace too small or misaligned");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int32_t* hist = reinterpret_cast<int32_t*>(partial + kMaxGroups);
  if (int rc = launch_counts(topk_ids, is_padding, rows, top_k, experts, false, counts, stats, hist, s)) return rc;
  const int groups = int(groups_of(rows));
  int rc = by_width(experts, scoring == 1, [&](auto per, auto sigmoid) {
    hipLaunchKernelGGL((loss_kernel<decltype(per)::value, decltype(sigmoid)::value>), dim3(unsigned(groups)), dim3(kThreads), 0, s,
                       logits, dtype, stride, is_padding, rows, int(experts), stats, partial);
  });
  if (rc) return rc;
  hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(64), 0, s, partial, groups, stats + experts, loss);
  return vq::check_launch("moe balance");
}

extern "C" int moe_balance_grad(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const uint8_t* is_padding,
                                int scoring, const float* stats, const float* upstream, void* grad, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, 1)) return rc;
  if (int rc = check_logits(logits, dtype, rows, experts, stride, scoring)) return rc;
  if (rows == 0) return vq::kOk;
  if (!stats || !upstream || !grad) return vq::fail("moe balance: null pointer");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned groups = unsigned(std::min<int64_t>((rows + kWaves - 1) / kWaves, 8 * kMaxGroups));
  return by_width(experts, scoring == 1, [&](auto per, auto sigmoid) {
    hipLaunchKernelGGL((grad_kernel<decltype(per)::value, decltype(sigmoid)::value>), dim3(groups), dim3(kThreads), 0, s, logits,
                       dtype, stride, is_padding, rows, int(experts), stats, upstream, grad);
  });
}

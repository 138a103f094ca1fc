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
// much).  A row whose logits leave nothing has p = 0: all of them -inf or, with
// sigmoids, below kNothing.  A p below 2^-66 may count as 0.  Counts are whole
// numbers, so their atomics give one result in any order; the rows' parts are
// summed in 64 bits in a fixed order.
//
// Bound by the logits' bytes where rows are many: at 65536 rows of 256 in FP32 (64
// MiB, 14 us at the rate of a large copy) the loss takes 17 us (sigmoids, with
// padding marked, 18) after a count of 6 to 7 us and before a finish of 4 us, the
// gradient (twice the bytes) 23 to 24 us; at 200 rows of 128 one launch each, which
// costs less than its call from the host.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <type_traits>

#include "../../include/vllm_mi355x.h"
#include "common.h"
#include "moe_logits.h"

namespace balance {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kCountThreads = 1024;
constexpr int kMaxExperts = 1024;
// Workgroups that count: the count and the loss that adds them up take 6.3 + 17.2 us
// at 65536 rows of 256 with 32, 10.0 + 16.9 us with 16 (the loss with 64: 25.1).
constexpr int kMaxParts = 32;
constexpr int kLossThreads = 1024, kLossWaves = kLossThreads / 64;
constexpr int kMaxGroups = 512;  // workgroups of the loss: two a CU, few enough to add up the counts
constexpr int kGradGroups = 2048;
// Calls of up to so many logits, whose rows a workgroup takes in up to so many steps
// (of one, two or four rows a wavefront), run in one workgroup and launch: a step
// costs 0.9 us, the launches of the others 12 whatever their rows.  In us, one workgroup
// and several: 512 rows of 8 12.1 and 12.7, 1024 18.9 and 12.7, 4096 59.7 and 12.7; 256
// rows of 128 11.4 and 11.8; 128 rows of 256 11.1 and 12.2.
constexpr int kOneLogits = 1 << 15;
constexpr int kOneSteps = 8;

// ---- a row of logits in the lanes of a wavefront (moe_logits.h) ---------------------

using logits::exp_nonpositive;
using logits::kLog2e;
using logits::lanes_max;
using logits::lanes_sum;
using logits::load_row;
using logits::product;
using logits::row_max;
using logits::Rows;
using logits::Shape;
using logits::Values;

using logits::kNothing;  // (a row whose logits all lie below it, masks among them, leaves nothing with sigmoids)

// A row's r from z = e^l / e^shift (softmax) or the sigmoid / 2^shift, and `sum`, z's
// sum (both in all its lanes); in place of the logits the slopes p (softmax) or p (1 -
// sigmoid).
template <typename S, bool kSigmoid>
__device__ __forceinline__ float shifted_terms(Values<S>& x, const float* f, int l, int lane, float shift, float& sum) {
  float dot = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) {
    typedef float f4_t __attribute__((ext_vector_type(4)));
    const f4_t w = *reinterpret_cast<const f4_t*>(f + 4 * (S::kLanes * i + l));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float z;
      if constexpr (kSigmoid) {
        const float a = x.v[i][j], u = exp_nonpositive(-fabsf(a), shift), t = __builtin_amdgcn_ldexpf(u, int(shift));
        // (the reciprocal of 1 .. 2 as the hardware rounds it, off by one step at most)
        const float large = __builtin_amdgcn_rcpf(1 + t), small = u * large;
        z = a >= 0 ? large : small;
        x.v[i][j] = large * small;
        if (a != a) z = x.v[i][j] = a;
      } else {
        z = x.v[i][j] = exp_nonpositive(x.v[i][j] - shift);
      }
      sum += z;
      dot = __builtin_fmaf(w[j], z, dot);
    }
  }
  sum = lanes_sum<S::kLanes>(sum, lane);
  dot = lanes_sum<S::kLanes>(dot, lane);
  const float inv = sum == 0 ? 0.0f : 1 / sum;
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[i][j] *= inv;
  return product(dot, inv);
}

// From a row's logits its r = sum f p (in all its lanes), and in place of the
// logits the slopes.  f: LDS, zeros past the last expert up to a whole step.
// again(): the logits once more.
template <typename S, bool kSigmoid, typename Again>
__device__ __forceinline__ float row_terms(Values<S>& x, const float* f, int l, int lane, const Again& again) {
  float sum;
  if constexpr (kSigmoid) {
    float r = shifted_terms<S, true>(x, f, l, lane, 0.0f, sum);
    // A row of tiny sigmoids alone (logits below -41) holds them over 2^k, about the
    // largest: p does not change by that, and none of weight is lost below 2^-126.
    // Such rows are read and computed again: 65536 of 256 cost the loss 41 us for 27, so
    // that rows in whose sums those below 2^-126 weigh nothing are left as they are;
    // their logits kept in registers would cost all rows a microsecond.
    const bool small = sum < 0x1p-60f;
    if (__builtin_expect(__any(small), 0)) {
      x = again();
      const float m = row_max(x, lane);
      const float k = small && m < 0 && m >= kNothing ? __builtin_ceilf(m * kLog2e) : 0.0f;
      r = shifted_terms<S, true>(x, f, l, lane, k, sum);
    }
    return r;
  } else {
    float m = row_max(x, lane);
    if (m == -__builtin_inff()) m = 0;
    return shifted_terms<S, false>(x, f, l, lane, m, sum);
  }
}

// ---- counts ---------------------------------------------------------------------------

struct Counting {
  const int32_t* ids;
  const uint8_t* padding;
  int64_t rows;
  int top_k, experts;
};

// count (LDS, experts + 1 zeros): the slots first, first + step, ... by expert, and at
// its end the rows that these begin.  Slot by slot, so that a wavefront's loads are of
// neighbours; eight slots at once, their loads on their way together.
__device__ __forceinline__ void count_slots(const Counting& g, int64_t first, int64_t step, int* count) {
  constexpr int kEach = 8;
  const int64_t slots = g.rows * g.top_k;
  int mine = 0;
  for (int64_t s0 = first; s0 < slots; s0 += kEach * step) {
    int id[kEach];
    uint32_t row[kEach];
    uint8_t mark[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const uint32_t s = uint32_t(min(s0 + u * step, slots - 1));  // (slots fit 31 bits)
      row[u] = s / uint32_t(g.top_k);
      id[u] = g.ids[s];
      mark[u] = 0;
    }
    if (g.padding) {
#pragma unroll
      for (int u = 0; u < kEach; ++u) mark[u] = g.padding[row[u]];
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const bool counted = s0 + u * step < slots && !mark[u];
      if (counted && id[u] >= 0 && id[u] < g.experts) atomicAdd(&count[id[u]], 1);
      mine += counted && row[u] * uint32_t(g.top_k) == uint32_t(s0 + u * step);
    }
  }
  if (mine) atomicAdd(&count[g.experts], mine);
}

// hist[part][E + 1]: the part's slots by expert, and its rows (an expert's parts in
// one line make the sums slower: the loss 21.2 us for 17.0).
__global__ __launch_bounds__(kCountThreads) void count_kernel(Counting g, int32_t* hist) {
  __shared__ int count[kMaxExperts + 1];
  for (int e = threadIdx.x; e <= g.experts; e += kCountThreads) count[e] = 0;
  __syncthreads();
  count_slots(g, int64_t(blockIdx.x) * kCountThreads + threadIdx.x, int64_t(gridDim.x) * kCountThreads, count);
  __syncthreads();
  for (int e = threadIdx.x; e <= g.experts; e += kCountThreads) hist[int64_t(blockIdx.x) * (g.experts + 1) + e] = count[e];
}

// The parts' sum for entry e, all its loads on their way at once (another XCD
// wrote them: a trip to memory).
__device__ __forceinline__ int64_t total_of(const int32_t* hist, int parts, int experts, int e) {
  int n[kMaxParts];
#pragma unroll
  for (int p = 0; p < kMaxParts; ++p) n[p] = hist[int64_t(min(p, parts - 1)) * (experts + 1) + e];
  int64_t sum = 0;
#pragma unroll
  for (int p = 0; p < kMaxParts; ++p) sum += p < parts ? n[p] : 0;
  return sum;
}

__global__ __launch_bounds__(kThreads) void totals_kernel(const int32_t* hist, int parts, int experts, bool add, int64_t* counts) {
  for (int e = threadIdx.x; e < experts; e += kThreads) {
    const int64_t c = total_of(hist, parts, experts, e);
    counts[e] = add ? counts[e] + c : c;
  }
}

// f_e of c slots, where n rows of top_k count.
__device__ __forceinline__ float share_of(int64_t c, int64_t n, int top_k, int experts) {
  return n ? float(double(c) * experts / (double(n) * top_k)) : 0.0f;
}

// ---- loss -------------------------------------------------------------------------------

// Rows first, first + step, ... of this wavefront (S::kRows at once): the sum of
// their r, in lane 0 of each row's lanes the row's own.
template <typename S, int kDtype, bool kSigmoid>
__device__ __forceinline__ double sum_rows(const Rows& g, int64_t first, int64_t step, const float* f, int lane) {
  const int l = lane % S::kLanes, sub = lane / S::kLanes;
  double sum = 0;
  if (first >= g.rows) return sum;
  // a row ahead: the next one's logits are on their way while this one's are used
  const auto row = [&](int64_t t) { return load_row<S, kDtype>(g, min(t, g.rows - 1), l); };
  const auto mark = [&](int64_t t) { return g.padding ? g.padding[min(t, g.rows - 1)] : uint8_t(0); };
  Values<S> next = row(first + sub);
  uint8_t next_mark = mark(first + sub);
  for (int64_t t = first + sub; t - sub < g.rows; t += step) {
    Values<S> x = next;
    const bool counted = t < g.rows && !next_mark;
    if (t - sub + step < g.rows) {
      next = row(t + step);
      next_mark = mark(t + step);
    }
    const float r = row_terms<S, kSigmoid>(x, f, l, lane, [&] { return row(t); });
    if (counted && l == 0) sum += r;
  }
  return sum;
}

// The sum over a workgroup's `waves` wavefronts, in order (part: as many entries).
__device__ __forceinline__ double block_sum(double v, double* part, int waves) {
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0;
  for (int w = 0; w < waves; ++w) sum += part[w];
  return sum;
}

struct Results {
  float* loss;
  int64_t* counts;
  float* stats;  // f_e, then 1 / n
};

// All of a small call in one workgroup.
template <typename S, int kDtype, bool kSigmoid>
__global__ __launch_bounds__(1024) void one_kernel(Rows g, Counting c, Results out) {
  __shared__ int count[kMaxExperts + 1];
  __shared__ __attribute__((aligned(16))) float f[kMaxExperts];
  __shared__ double part[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  for (int e = tid; e <= c.experts; e += 1024) count[e] = 0;
  __syncthreads();
  count_slots(c, tid, 1024, count);
  __syncthreads();
  const int n = count[c.experts];
  for (int e = tid; e < kMaxExperts; e += 1024) {
    f[e] = e < c.experts ? share_of(count[e], n, c.top_k, c.experts) : 0.0f;
    if (e < c.experts) {
      out.counts[e] = count[e];
      out.stats[e] = f[e];
    }
  }
  if (tid == 0) out.stats[c.experts] = n ? float(1.0 / double(n)) : 0.0f;
  __syncthreads();
  const double sum = block_sum(sum_rows<S, kDtype, kSigmoid>(g, wave * S::kRows, 16 * S::kRows, f, lane), part, 16);
  if (tid == 0) out.loss[0] = n ? float(sum / double(n)) : 0.0f;
}

// partial[workgroup] = the sum of its rows' r.  Every workgroup adds up the parts'
// counts for itself, an entry a thread (one thread the rows': as many requests to
// the same lines as there are wavefronts would queue up in L2).  A launch of its
// own finishes: 512 arrivals at one counter took 10 us.
template <typename S, int kDtype, bool kSigmoid>
__global__ __launch_bounds__(kLossThreads) void loss_kernel(Rows g, int top_k, const int32_t* hist, int parts, double* partial) {
  __shared__ __attribute__((aligned(16))) float f[kMaxExperts];
  __shared__ double part[kLossWaves];
  __shared__ int64_t counted;
  static_assert(kMaxExperts <= kLossThreads, "a thread an expert");
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  const int64_t mine = tid < g.experts ? total_of(hist, parts, g.experts, tid) : 0;
  if (tid == kLossThreads - 1) counted = total_of(hist, parts, g.experts, g.experts);
  __syncthreads();
  if (tid < S::kLanes * S::kSteps * 4) f[tid] = tid < g.experts ? share_of(mine, counted, top_k, g.experts) : 0.0f;
  __syncthreads();
  const int64_t first = (int64_t(blockIdx.x) * kLossWaves + wave) * S::kRows;
  const double sum = block_sum(sum_rows<S, kDtype, kSigmoid>(g, first, int64_t(gridDim.x) * kLossWaves * S::kRows, f, lane), part, kLossWaves);
  if (tid == 0) partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kLossThreads) void finish_kernel(const double* partial, int groups, const int32_t* hist, int parts,
                                                              int experts, int top_k, Results out) {
  __shared__ double part[kLossWaves];
  __shared__ int64_t counted;
  static_assert(kMaxGroups <= kLossThreads, "a thread a workgroup's sum");
  const int tid = threadIdx.x;
  const double one = tid < groups ? partial[tid] : 0.0;
  const int64_t mine = tid < experts ? total_of(hist, parts, experts, tid) : 0;
  if (tid == kLossThreads - 1) counted = total_of(hist, parts, experts, experts);
  const double all = block_sum(one, part, kLossWaves);
  const int64_t n = counted;
  if (tid < experts) {
    out.counts[tid] = mine;
    out.stats[tid] = share_of(mine, n, top_k, experts);
  }
  if (tid == 0) {
    out.loss[0] = n ? float(all / double(n)) : 0.0f;
    out.stats[experts] = n ? float(1.0 / double(n)) : 0.0f;
  }
}

template <typename S, int kDtype, bool kSigmoid>
__global__ __launch_bounds__(kThreads) void grad_kernel(Rows g, const float* stats, const float* upstream, void* grad) {
  __shared__ __attribute__((aligned(16))) float f[kMaxExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  const int l = lane % S::kLanes, sub = lane / S::kLanes;
  for (int e = tid; e < S::kLanes * S::kSteps * 4; e += kThreads) f[e] = e < g.experts ? stats[e] : 0.0f;
  __syncthreads();
  const float scale = upstream[0] * stats[g.experts];
  // (rows of the gradient lie close: on whole fours where the experts do)
  const bool wide = g.experts % 4 == 0;
  for (int64_t t0 = (int64_t(blockIdx.x) * kWaves + wave) * S::kRows; t0 < g.rows; t0 += int64_t(gridDim.x) * kWaves * S::kRows) {
    const int64_t t = t0 + sub;
    const bool counted = t < g.rows && !(g.padding && g.padding[min(t, g.rows - 1)]);
    const auto row = [&] { return load_row<S, kDtype>(g, t < g.rows ? t : g.rows - 1, l); };
    Values<S> x = row();
    const float r = row_terms<S, kSigmoid>(x, f, l, lane, row);
    if (t >= g.rows) continue;
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      const int e = 4 * (S::kLanes * i + l);
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = counted ? scale * x.v[i][j] * (f[e + j] - r) : 0.0f;
      const int64_t at = t * g.experts + e;
      if (wide && e < g.experts) {
        if constexpr (kDtype == vq::kFP32) {
          typedef float f4_t __attribute__((ext_vector_type(4)));
          *reinterpret_cast<f4_t*>(static_cast<float*>(grad) + at) = f4_t{v[0], v[1], v[2], v[3]};
        } else {
          typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
          const auto half = [](float a) {
            return uint32_t(kDtype == vq::kBF16 ? vq::f32_to_bf16(a) : __builtin_bit_cast(uint16_t, _Float16(a)));
          };
          *reinterpret_cast<u2_t*>(static_cast<uint16_t*>(grad) + at) = u2_t{half(v[0]) | (half(v[1]) << 16), half(v[2]) | (half(v[3]) << 16)};
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (e + j < g.experts) vq::store_act(grad, kDtype, at + j, v[j]);
        }
      }
    }
  }
}

// launch(shape, dtype, sigmoid) with the call's as types.
template <typename F>
int dispatch(int64_t experts, int dtype, bool sigmoid, const F& launch) {
  const auto shaped = [&](auto shape) {
    const auto typed = [&](auto type) {
      if (sigmoid) launch(shape, type, std::true_type{});
      else launch(shape, type, std::false_type{});
    };
    if (dtype == vq::kBF16) typed(std::integral_constant<int, vq::kBF16>{});
    else if (dtype == vq::kFP16) typed(std::integral_constant<int, vq::kFP16>{});
    else typed(std::integral_constant<int, vq::kFP32>{});
  };
  if (experts <= 64) shaped(Shape<16, 1>{});
  else if (experts <= 128) shaped(Shape<32, 1>{});
  else if (experts <= 256) shaped(Shape<64, 1>{});
  else if (experts <= 512) shaped(Shape<64, 2>{});
  else shaped(Shape<64, 4>{});
  return vq::check_launch("moe balance");
}

int rows_at_once(int64_t experts) { return experts <= 64 ? 4 : experts <= 128 ? 2 : 1; }
int64_t parts_of(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(kMaxParts, (rows + 255) / 256)); }
int64_t groups_of(int64_t rows, int64_t experts, int64_t waves, int64_t most) {
  const int64_t each = waves * rows_at_once(experts);
  return std::max<int64_t>(1, std::min<int64_t>(most, (rows + each - 1) / each));
}

int check_sizes(int64_t rows, int64_t experts, int64_t top_k) {
  if (rows < 0 || rows > INT_MAX) return vq::fail("moe balance: rows out of range");
  if (experts <= 0 || experts > kMaxExperts) return vq::fail("moe balance: between 1 and 1024 experts");
  if (top_k <= 0 || top_k > INT_MAX || rows * top_k > INT_MAX) return vq::fail("moe balance: top_k out of range");
  return vq::kOk;
}

// The workspace: partial sums, then the parts' histograms.
struct Workspace {
  double* partial;
  int32_t* hist;
  static int64_t bytes(int64_t experts) { return kMaxGroups * 8 + kMaxParts * (experts + 1) * 4; }
  explicit Workspace(void* base)
      : partial(static_cast<double*>(base)), hist(reinterpret_cast<int32_t*>(partial + kMaxGroups)) {}
};

int launch_count(const Counting& c, const Workspace& w, hipStream_t s) {
  hipLaunchKernelGGL(count_kernel, dim3(unsigned(parts_of(c.rows))), dim3(kCountThreads), 0, s, c, w.hist);
  return vq::check_launch("moe counts");
}

Rows rows_of(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const uint8_t* padding) {
  const int64_t four = 4 * vq::dtype_bytes(dtype);
  const bool wide = experts % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % four == 0;
  return {logits, stride, padding, rows, int(experts), wide};
}

int check_logits(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, int scoring) {
  if (dtype != vq::kBF16 && dtype != vq::kFP16 && dtype != vq::kFP32) return vq::fail("moe balance: logits must be BF16, FP16 or FP32");
  if (scoring != 0 && scoring != 1) return vq::fail("moe balance: scoring must be softmax (0) or sigmoid (1)");
  if (stride < 0 || (rows > 1 && stride < experts) || stride > (int64_t(1) << 31)) return vq::fail("moe balance: row stride out of range");
  if (rows > 0 && !logits) return vq::fail("moe balance: null pointer");
  return vq::kOk;
}

bool aligned8(const void* p) { return reinterpret_cast<uintptr_t>(p) % 8 == 0; }

// A call's arrays: no output may overlap another array, and each lies on its elements.
struct Span {
  const void* p;
  int64_t bytes, element;
};
int check_spans(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  for (const Span* a = outputs.begin(); a != outputs.end(); ++a) {
    for (const Span* b = outputs.begin(); b != a; ++b) {
      if (vq::overlaps(a->p, a->bytes, b->p, b->bytes)) return vq::fail("moe balance: arguments must not overlap");
    }
    for (const Span& b : inputs) {
      if (vq::overlaps(a->p, a->bytes, b.p, b.bytes)) return vq::fail("moe balance: arguments must not overlap");
    }
  }
  for (const auto* list : {&outputs, &inputs}) {
    for (const Span& a : *list) {
      if (reinterpret_cast<uintptr_t>(a.p) % uintptr_t(a.element)) return vq::fail("moe balance: misaligned pointer");
    }
  }
  return vq::kOk;
}

// Bytes from the first logit to the last.
int64_t logits_bytes(int dtype, int64_t rows, int64_t experts, int64_t stride) {
  return rows > 0 ? ((rows - 1) * stride + experts) * vq::dtype_bytes(dtype) : 0;
}

}  // namespace
}  // namespace balance

extern "C" int64_t moe_balance_workspace_size(int64_t rows, int64_t experts) {
  using namespace balance;
  if (check_sizes(rows, experts, 1)) return -1;
  return Workspace::bytes(experts);
}

extern "C" int moe_expert_counts(const int32_t* topk_ids, const uint8_t* is_padding, int64_t rows, int64_t top_k, int64_t experts,
                                 int add, int64_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, top_k)) return rc;
  if (!counts || !workspace || (rows > 0 && !topk_ids)) return vq::fail("moe balance: null pointer");
  if (workspace_bytes < Workspace::bytes(experts) || !aligned8(workspace)) return vq::fail("moe balance: workspace too small or misaligned");
  if (int rc = check_spans({{counts, experts * 8, 8}, {workspace, Workspace::bytes(experts), 8}},
                           {{topk_ids, rows * top_k * 4, 4}, {is_padding, rows, 1}})) {
    return rc;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Workspace w(workspace);
  if (int rc = launch_count({topk_ids, is_padding, rows, int(top_k), int(experts)}, w, s)) return rc;
  hipLaunchKernelGGL(totals_kernel, dim3(1), dim3(kThreads), 0, s, w.hist, int(parts_of(rows)), int(experts), add != 0, counts);
  return vq::check_launch("moe counts");
}

extern "C" int moe_balance_loss(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const int32_t* topk_ids,
                                int64_t top_k, const uint8_t* is_padding, int scoring, float* loss, int64_t* counts, float* stats,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, top_k)) return rc;
  if (int rc = check_logits(logits, dtype, rows, experts, stride, scoring)) return rc;
  if (!loss || !counts || !stats || !workspace || (rows > 0 && !topk_ids)) return vq::fail("moe balance: null pointer");
  if (workspace_bytes < Workspace::bytes(experts) || !aligned8(workspace)) return vq::fail("moe balance: workspace too small or misaligned");
  if (int rc = check_spans({{loss, 4, 4}, {counts, experts * 8, 8}, {stats, (experts + 1) * 4, 4}, {workspace, Workspace::bytes(experts), 8}},
                           {{logits, logits_bytes(dtype, rows, experts, stride), vq::dtype_bytes(dtype)},
                            {topk_ids, rows * top_k * 4, 4}, {is_padding, rows, 1}})) {
    return rc;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Counting c{topk_ids, is_padding, rows, int(top_k), int(experts)};
  const Rows g = rows_of(logits, dtype, rows, experts, stride, is_padding);
  const Results out{loss, counts, stats};
  if (rows * experts <= kOneLogits && rows <= kOneSteps * 16 * rows_at_once(experts)) {
    return dispatch(experts, dtype, scoring == 1, [&](auto shape, auto type, auto sigmoid) {
      hipLaunchKernelGGL((one_kernel<decltype(shape), decltype(type)::value, decltype(sigmoid)::value>), dim3(1), dim3(1024), 0, s, g, c, out);
    });
  }
  const Workspace w(workspace);
  if (int rc = launch_count(c, w, s)) return rc;
  const unsigned groups = unsigned(groups_of(rows, experts, kLossWaves, kMaxGroups));
  const int parts = int(parts_of(rows));
  const int rc = dispatch(experts, dtype, scoring == 1, [&](auto shape, auto type, auto sigmoid) {
    hipLaunchKernelGGL((loss_kernel<decltype(shape), decltype(type)::value, decltype(sigmoid)::value>), dim3(groups), dim3(kLossThreads), 0,
                       s, g, int(top_k), w.hist, parts, w.partial);
  });
  if (rc) return rc;
  hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(kLossThreads), 0, s, w.partial, int(groups), w.hist, parts, int(experts), int(top_k), out);
  return vq::check_launch("moe balance");
}

extern "C" int moe_balance_grad(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const uint8_t* is_padding,
                                int scoring, const float* stats, const float* upstream, void* grad, void* stream) {
  using namespace balance;
  if (int rc = check_sizes(rows, experts, 1)) return rc;
  if (int rc = check_logits(logits, dtype, rows, experts, stride, scoring)) return rc;
  if (rows == 0) return vq::kOk;
  if (!stats || !upstream || !grad) return vq::fail("moe balance: null pointer");
  if (reinterpret_cast<uintptr_t>(grad) % (4 * vq::dtype_bytes(dtype))) return vq::fail("moe balance: grad must be aligned to four elements");
  // (in place of contiguous logits a row is read whole before it is written)
  const bool in_place = grad == logits && (rows == 1 || stride == experts);
  if (int rc = check_spans({{grad, rows * experts * vq::dtype_bytes(dtype), 1}},
                           {{in_place ? nullptr : logits, logits_bytes(dtype, rows, experts, stride), 1}, {is_padding, rows, 1},
                            {stats, (experts + 1) * 4, 4}, {upstream, 4, 4}})) {
    return rc;
  }
  if (reinterpret_cast<uintptr_t>(logits) % uintptr_t(vq::dtype_bytes(dtype))) return vq::fail("moe balance: misaligned pointer");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Rows g = rows_of(logits, dtype, rows, experts, stride, is_padding);
  const unsigned groups = unsigned(groups_of(rows, experts, kWaves, kGradGroups));
  return dispatch(experts, dtype, scoring == 1, [&](auto shape, auto type, auto sigmoid) {
    hipLaunchKernelGGL((grad_kernel<decltype(shape), decltype(type)::value, decltype(sigmoid)::value>), dim3(groups), dim3(kThreads), 0, s,
                       g, stats, upstream, grad);
  });
}

// Routing from a router's logits: the experts of each row, by groups where asked, and
// their weights, with the weights' gradient.
//
// s_e is the softmax or the sigmoid of the row's logit l_e, the key of an expert its
// score plus its bias; without a bias the logit orders as its score does and is the
// key.  A group of consecutive experts scores its largest key, with a bias its two
// largest's sum; the best groups stay open, and of their experts the best are chosen,
// always the lower number of equals.  Over the chosen (c the scale)
//
//   w_j = c s_j, or renormalized c s_j / S, S their sum,
//
// and with g the weights' gradient, the choice constant, d_e = dL/dl_e:
//
//   softmax, renormalized:  w_e (g_e - sum_j w_j g_j / sum_j w_j)            of chosen experts
//   sigmoid, renormalized:  w_e (1 - s_e) (g_e - sum_j w_j g_j / sum_j w_j)
//   sigmoid:                w_e (1 - s_e) g_e
//   softmax:                [chosen] w_e g_e - s_e sum_j w_j g_j     of all experts.
//
// An expert is masked, and not chosen, where its score is below 2^-1022 of the
// largest possible (logits 708.396 below 0 or, for softmax, the row's largest; -inf
// among them) or its bias is -inf or NaN.  Slots left over hold -1 and weight 0.  A row
// with a NaN (softmax: or +inf) has weights NaN, its experts chosen without that one.
//
// Keys with a bias are FP32 sums, off by up to 2^-20; where two that decide the
// choice or its order lie closer than their errors, the wavefront's rows are keyed and
// chosen again in 64 bits, so that the choice is always that of 64-bit keys.  Equal keys are
// among these: rare with a bias of any values, but 16-bit logits with a bias of zeros often
// tie (65536 rows of 256 in BF16, four of eight groups: 153 us for 59, without groups 111
// for 43; FP32 logits 59 and 42).  Without a bias there is no second choice (31 and 22).
//
// What bounds it: few rows, the launch (1 row of 256, eight groups: 5.2 us on the GPU, 7.4 a
// call); many, vector instructions: 65536 rows of 256 FP32 logits, sigmoid, bias, four of eight
// groups open, take 57 us forward (67 MB at 1.2 TB/s: the sigmoids and the selection) and 15
// back (the gradient's stores, 67 MB at 4.5 TB/s).  More than 256 experts have 32 lanes a row and a
// scan of all keys a slot: 65536 rows of 384 87 us, of 512 91 (without a bias 64 both).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <type_traits>

#include "../../include/vllm_mi355x.h"
#include "common.h"
#include "moe_logits.h"

namespace route {
namespace {

using logits::exp_nonpositive;
using logits::kLog2e;
using logits::kNothing;
using logits::lanes_max;
using logits::lanes_sum;
using logits::load_row;
using logits::Rows;
using logits::Shape;
using logits::Values;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kMaxSlots = 64;   // a lane a slot
constexpr int kMaxGroups = 64;  // a bit a group
constexpr unsigned kMaxGrid = 1024;  // four workgroups a CU, as many as are at work

struct Choice {
  const float* bias;
  int top_k, groups, topk_groups;  // groups 1: none
  int group_experts;
  int group_lanes;  // lanes that hold a group in one step, a power of two; 0: groups lie otherwise
  bool renormalize;
  float scale;
  float* weights;
  int32_t* ids;
};

__device__ __forceinline__ float minus_inf() { return -__builtin_inff(); }

// Keys are compared as whole numbers of FP32's order (whose maxima take one instruction
// across lanes; a float's are quieted first).  Both zeros are one.
__device__ __forceinline__ int ordered(float v) {
  const int b = __builtin_bit_cast(int, v + 0.0f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int v) { return __builtin_bit_cast(float, v ^ ((v >> 31) & 0x7fffffff)); }
constexpr int kNone = int(0x807fffffu);  // -inf

// v from the lane kTurn places before in the row of 16 lanes, from its first ones on the last.
template <int kTurn>
__device__ __forceinline__ int turned(int v) {
  return __builtin_amdgcn_mov_dpp(v, 0x120 | kTurn, 0xF, 0xF, false);  // row_ror
}
template <int kTurn = 1, typename F>
__device__ __forceinline__ void each_turn(const F& f) {
  if constexpr (kTurn < 16) {
    f(std::integral_constant<int, kTurn>{});
    each_turn<kTurn + 1>(f);
  }
}
template <int d>
__device__ __forceinline__ int xor_int(int v, int lane) {
  if constexpr (d == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false);  // row_half_mirror: lane ^ 7
  else return __builtin_bit_cast(int, vq::xor_lanes<d>(__builtin_bit_cast(float, v), lane));
}
// f over a row's lanes.
template <int kLanes, typename F>
__device__ __forceinline__ int over_lanes(int v, int lane, const F& f) {
  if constexpr (kLanes > 32) v = f(v, xor_int<32>(v, lane));
  if constexpr (kLanes > 16) v = f(v, xor_int<16>(v, lane));
  v = f(v, turned<8>(v));
  v = f(v, turned<4>(v));
  v = f(v, turned<2>(v));
  return f(v, turned<1>(v));
}
template <int kLanes>
__device__ __forceinline__ int most(int v, int lane) { return over_lanes<kLanes>(v, lane, [](int a, int b) { return max(a, b); }); }
template <int kLanes>
__device__ __forceinline__ int least(int v, int lane) { return over_lanes<kLanes>(v, lane, [](int a, int b) { return min(a, b); }); }
template <int kLanes>
__device__ __forceinline__ double lanes_max(double v) {
#pragma unroll
  for (int d = kLanes / 2; d > 0; d /= 2) v = fmax(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ int larger(int a, int b) { return max(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ int smaller(int a, int b) { return min(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }

// The two largest of a run of keys.
template <typename Key>
struct Top2 {
  Key first, second;
  __device__ __forceinline__ void add(Key k) {
    second = larger(second, smaller(first, k));
    first = larger(first, k);
  }
  // with the lanes' d places on, where those between have joined (whichever of these)
  template <int d>
  __device__ __forceinline__ void join(int lane) {
    const Key a = xor_int<d>(first, lane), b = xor_int<d>(second, lane);
    second = larger(smaller(first, a), larger(second, b));
    first = larger(first, a);
  }
};

// What lies in LDS: the wavefront's rows of keys, and for groups that do not fill whole
// lanes of a step the groups of four neighbouring experts, a byte each.
template <typename S>
struct KeySpace {
  static constexpr int kPadded = 4 * S::kLanes * S::kSteps;
  double* keys;            // [kRows][kPadded], those of 32 bits in its first half
  const uint32_t* group4;  // [kPadded / 4]
  uint16_t* list;          // [64]: a place a lane

  template <typename Key>
  __device__ __forceinline__ Key* row(int lane) const {
    return reinterpret_cast<Key*>(keys) + (lane / S::kLanes) * kPadded;
  }
};

// LDS of one wavefront's own: what its lanes have written, its lanes may read.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Keys of closed groups become -inf.  error: what a key may be off by at most, apart from its
// own rounding; doubt: set where it may decide.
template <typename S, bool kTwo>
__device__ __forceinline__ void close_groups(int (&key)[S::kSteps][4], const Choice& c, const KeySpace<S>& space, int l, int lane,
                                             float error, bool& doubt) {
  const bool in_lanes = c.group_lanes > 0;
  int score[S::kSteps];
  float size = 0;  // of the keys that scores are made of
  const auto finish = [&](const Top2<int>& t) {
    if constexpr (!kTwo) return t.first;
    const float a = value_of(t.first), b = value_of(t.second), m = fmaxf(fabsf(a), b > minus_inf() ? fabsf(b) : 0.0f);
    size = fmaxf(size, m < __builtin_inff() ? m : 0.0f);
    return ordered(b > minus_inf() ? a + b : a);
  };
  const int shift = in_lanes ? __builtin_ctz(c.group_lanes) : 0;
  const auto group_at = [&](int i) { return in_lanes ? (S::kLanes * i + l) >> shift : l; };
  if (in_lanes) {
    Top2<int> t[S::kSteps];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      t[i] = {key[i][0], kNone};
#pragma unroll
      for (int j = 1; j < 4; ++j) t[i].add(key[i][j]);
    }
    const auto join = [&](auto d) {
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i) t[i].template join<decltype(d)::value>(lane);
    };
    if (c.group_lanes > 1) join(std::integral_constant<int, 1>{});
    if (c.group_lanes > 2) join(std::integral_constant<int, 2>{});
    if (c.group_lanes > 4) join(std::integral_constant<int, 4>{});
    if (c.group_lanes > 8) join(std::integral_constant<int, 8>{});
    if constexpr (S::kLanes > 16) {
      if (c.group_lanes > 16) join(std::integral_constant<int, 16>{});
    }
    if constexpr (S::kLanes > 32) {
      if (c.group_lanes > 32) join(std::integral_constant<int, 32>{});
    }
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) score[i] = finish(t[i]);
  } else {
    // lane g takes group g, its keys from LDS (each lane from a place of its own on)
    int* row = space.template row<int>(lane);
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) row[4 * (S::kLanes * i + l) + j] = key[i][j];
    wave_lds_fence();
    Top2<int> t{kNone, kNone};
    if (l < c.groups) {
      int at = l % c.group_experts;
      for (int n = 0; n < c.group_experts; ++n) {
        t.add(row[l * c.group_experts + at]);
        at = at + 1 == c.group_experts ? 0 : at + 1;
      }
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) score[i] = kNone;
    score[0] = finish(t);
  }
  float tolerance = 0;
  if constexpr (kTwo) {
    // four keys decide between two scores, each off by its error and half a step
    // (sizes are not negative: they order as their bits)
    tolerance = 4 * error + value_of(most<S::kLanes>(ordered(size), lane)) * 0x1p-21f;
  }
  uint64_t open = 0;
  int last = kNone;
  for (int q = 0;; ++q) {
    int m = score[0];
#pragma unroll
    for (int i = 1; i < S::kSteps; ++i) m = max(m, score[i]);
    m = most<S::kLanes>(m, lane);
    if (q == c.topk_groups) {
      if constexpr (kTwo) doubt = doubt || value_of(last) - value_of(m) <= tolerance;
      break;
    }
    int g = INT_MAX;
#pragma unroll
    for (int i = S::kSteps - 1; i >= 0; --i) g = score[i] == m ? group_at(i) : g;
    g = least<S::kLanes>(g, lane);
    if (m > kNone) open |= uint64_t(1) << (g & 63);
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) score[i] = group_at(i) == g ? kNone : score[i];
    last = m;
  }
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) {
    if (in_lanes) {
      const bool kept = (open >> (group_at(i) & 63)) & 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) key[i][j] = kept ? key[i][j] : kNone;
    } else {
      const uint32_t four = space.group4[S::kLanes * i + l];
#pragma unroll
      for (int j = 0; j < 4; ++j) key[i][j] = (open >> (four >> (8 * j) & 63)) & 1 ? key[i][j] : kNone;
    }
  }
}

// The same as choose (below) for rows of 16 lanes and up to 15 slots, where few enough keys
// come into question, else false: those not below the `need`th of the lanes' two largest each,
// which `need` keys at least are not.  They go to a lane each, 16 at most, which counts
// the better ones.  (By the largest of each lane alone one row in eight had more than 16.)
template <typename S, bool kBias>
__device__ __forceinline__ bool choose_ranked(const int (&key)[S::kSteps][4], const Choice& c, const KeySpace<S>& space, int l, int lane,
                                              float error, bool& doubt, int& mine) {
  static_assert(S::kLanes == 16 && S::kSteps <= 4, "rows of 16 lanes");
  const int need = c.top_k + (kBias ? 1 : 0);
  int* row = space.template row<int>(lane);
  wave_lds_fence();
  Top2<int> t{key[0][0], kNone};
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) {
    typedef int i4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<i4_t*>(row + 4 * (16 * i + l)) = i4_t{key[i][0], key[i][1], key[i][2], key[i][3]};
#pragma unroll
    for (int j = i == 0; j < 4; ++j) t.add(key[i][j]);
  }
  // (lanes with equal ones go on together: the border is no higher for it)
  int border = kNone;
#pragma unroll 1
  for (int k = 0; k < need; ++k) {
    border = most<16>(t.first, lane);
    const bool gone = t.first == border;
    t.first = gone ? t.second : t.first;
    t.second = gone ? kNone : t.second;
  }
  uint32_t marks = 0;  // bit 4 i + j: key[i][j] comes into question
#pragma unroll
  for (int i = S::kSteps - 1; i >= 0; --i)
#pragma unroll
    for (int j = 3; j >= 0; --j) marks = 2 * marks + (key[i][j] >= border ? 1 : 0);
  // (the lanes' before this one's and its own, and all)
  const int count = __builtin_popcount(marks);
  int sum = count;
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xF, 0xF, true);  // row_shr
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xF, 0xF, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xF, 0xF, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xF, 0xF, true);
  const int total = most<16>(sum, lane);
  if (__any(total > 16)) return false;
  uint16_t* list = space.list + (lane & 48);
  for (int at = sum - count; __any(marks != 0); ++at) {
    if (marks) {
      const int bit = __builtin_ctz(marks);
      list[at] = uint16_t(4 * (16 * (bit >> 2) + l) + (bit & 3));
      marks &= marks - 1;
    }
  }
  wave_lds_fence();
  const int e = l < total ? list[l] : 0;
  const int k = l < total ? row[e] : kNone;
  // of equals the lower expert's
  const uint64_t place = l < total ? uint64_t(uint32_t(k) ^ 0x80000000u) << 32 | ~uint32_t(e) : 0;
  int rank = 0;
  each_turn([&](auto turn) {
    constexpr int n = decltype(turn)::value;
    const uint64_t other = uint64_t(uint32_t(turned<n>(int(place >> 32)))) << 32 | uint32_t(turned<n>(int(place)));
    rank += other > place;
  });
  const int to = 4 * ((lane & 48) | (l < total ? rank : 15));
  // (of lanes without a key the last lane may hear, where there is none better)
  const int sorted = __builtin_amdgcn_ds_permute(to, l < total ? e : -1);
  int best = __builtin_amdgcn_ds_permute(to, k);
  if (l >= total) best = kNone;
  if constexpr (kBias) {
    const float own = value_of(best), next = value_of(turned<15>(best));
    const bool close = l < c.top_k && own - next <= 2 * error + fabsf(own) * 0x1p-22f;
    const uint64_t any = __ballot(close);
    doubt = doubt || ((any >> (lane & 48)) & 0xffff) != 0;
  }
  mine = l < c.top_k && best > kNone ? sorted : -1;
  return true;
}

// Slot l's expert, or -1, in lane l of the row's lanes; the keys are used up.
template <typename S, bool kBias>
__device__ __forceinline__ int choose(int (&key)[S::kSteps][4], const Choice& c, const KeySpace<S>& space, int l, int lane, float error,
                                      bool& doubt) {
  if (c.groups > 1) close_groups<S, kBias>(key, c, space, l, lane, error, doubt);
  int mine = -1;
  if constexpr (S::kLanes == 16) {
    if (c.top_k < 16 && choose_ranked<S, kBias>(key, c, space, l, lane, error, doubt, mine)) return mine;
  }
  float last = 0;
  for (int k = 0;; ++k) {
    if (!kBias && k == c.top_k) break;
    int m = key[0][0];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max(m, key[i][j]);
    m = most<S::kLanes>(m, lane);
    if constexpr (kBias) {
      // (both off by their errors and half a step)
      doubt = doubt || (k > 0 && last - value_of(m) <= 2 * error + fabsf(last) * 0x1p-22f);
      if (k == c.top_k) break;
      last = value_of(m);
    }
    int e = INT_MAX;
#pragma unroll
    for (int i = S::kSteps - 1; i >= 0; --i)
#pragma unroll
      for (int j = 3; j >= 0; --j) e = key[i][j] == m ? 4 * S::kLanes * i + j : e;
    e = least<S::kLanes>(e == INT_MAX ? e : e + 4 * l, lane);
    if (l == k && m > kNone) mine = e;
    const int here = e - 4 * l;
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) key[i][j] = here == 4 * S::kLanes * i + j ? kNone : key[i][j];
  }
  return mine;
}

// The same from 64-bit keys in LDS (-inf: not to be chosen), which are used up.  In loops, so
// that it costs the rows without doubt no registers.
template <typename S>
__device__ __forceinline__ int choose_exact(double* row, const Choice& c, int experts, int l) {
  const double none = -__builtin_inf();
  wave_lds_fence();
  if (c.groups > 1) {
    Top2<double> t{none, none};
    if (l < c.groups) {
#pragma unroll 1
      for (int n = 0; n < c.group_experts; ++n) t.add(row[l * c.group_experts + n]);
    }
    double score = t.second > none ? t.first + t.second : t.first;
    uint64_t open = 0;
#pragma unroll 1
    for (int q = 0; q < c.topk_groups; ++q) {
      const double m = lanes_max<S::kLanes>(score);
      const int g = least<S::kLanes>(score == m ? l : INT_MAX, threadIdx.x & 63);
      if (m > none) open |= uint64_t(1) << (g & 63);
      score = l == g ? none : score;
    }
#pragma unroll 1
    for (int e = l; e < experts; e += S::kLanes) {
      if (!((open >> (e / c.group_experts)) & 1)) row[e] = none;
    }
    wave_lds_fence();
  }
  int mine = -1;
#pragma unroll 1
  for (int k = 0; k < c.top_k; ++k) {
    double best = none;
    int at = INT_MAX;
#pragma unroll 1
    for (int e = l; e < experts; e += S::kLanes) {  // (its lowest of equals)
      const double v = row[e];
      at = v > best ? e : at;
      best = fmax(best, v);
    }
    const double m = lanes_max<S::kLanes>(best);
    const int e = least<S::kLanes>(best == m ? at : INT_MAX, threadIdx.x & 63);
    if (l == k && m > none) mine = e;
    if (m > none && at == e) row[e] = none;
    wave_lds_fence();
  }
  return mine;
}

// 1 / (1 + e^-x), off by 2^-21 (whatever e^-x is off by times |x|, its part is small there).
__device__ __forceinline__ float sigmoid_key(float x) { return __builtin_amdgcn_rcpf(1 + __builtin_amdgcn_exp2f(x * -kLog2e)); }

// The same, off by 2^-21 of it.
__device__ __forceinline__ float sigmoid_of(float x) {
  const float u = exp_nonpositive(-fabsf(x)), large = __builtin_amdgcn_rcpf(1 + u);
  return x >= 0 ? large : u * large;
}

template <typename S, int kDtype, bool kSigmoid, bool kBias>
__global__ __launch_bounds__(kThreads, 4) void choose_kernel(Rows g, Choice c) {
  constexpr int kPadded = KeySpace<S>::kPadded;
  __shared__ __attribute__((aligned(16))) float bias[kBias ? kPadded : 4];
  __shared__ uint32_t group4[kPadded / 4];
  __shared__ __attribute__((aligned(16))) double rows[kWaves][S::kRows * kPadded];
  __shared__ uint16_t lists[kWaves][64];
  typedef float f4_t __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  const int l = lane % S::kLanes, sub = lane / S::kLanes;
  if constexpr (kBias) {
    for (int e = tid; e < kPadded; e += kThreads) bias[e] = e < g.experts ? c.bias[e] : minus_inf();
  }
  if (c.groups > 1 && !c.group_lanes) {
    for (int q = tid; q < kPadded / 4; q += kThreads) {
      uint32_t four = 0;
      for (int j = 0; j < 4; ++j) four |= uint32_t(min((4 * q + j) / c.group_experts, c.groups - 1)) << (8 * j);
      group4[q] = four;
    }
  }
  __syncthreads();
  const KeySpace<S> space{rows[wave], group4, lists[wave]};
  const int64_t step = int64_t(gridDim.x) * kWaves * S::kRows;
  const int64_t first = (int64_t(blockIdx.x) * kWaves + wave) * S::kRows;
  if (first >= g.rows) return;
  // a row ahead: the next one's logits are on their way while this one's are used
  const auto row = [&](int64_t t) { return load_row<S, kDtype>(g, min(t, g.rows - 1), l); };
  const auto mark = [&](int64_t t) { return g.padding ? g.padding[min(t, g.rows - 1)] : uint8_t(0); };
  Values<S> next = row(first + sub);
  uint8_t next_mark = mark(first + sub);
  for (int64_t t = first + sub; t - sub < g.rows; t += step) {
    Values<S> x = next;
    const bool padding = next_mark;
    if (t - sub + step < g.rows) {
      next = row(t + step);
      next_mark = mark(t + step);
    }
    // what poisons a row becomes -inf
    bool bad = false;
    float largest = minus_inf();
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& v = x.v[i][j];
        const bool b = kSigmoid ? v != v : !(v < __builtin_inff());
        bad |= b;
        v = b ? minus_inf() : v;
        if (!kSigmoid) largest = fmaxf(largest, v);
      }
    const uint64_t bads = __ballot(bad);
    const bool poisoned = (S::kLanes == 64 ? bads : (bads >> (S::kLanes * sub)) & ((uint64_t(1) << (S::kLanes & 63)) - 1)) != 0;
    float lowest = kNothing;  // logits from here on count
    if constexpr (!kSigmoid) {
      largest = lanes_max<S::kLanes>(largest, lane);
      if (largest == minus_inf()) largest = 0;
      lowest = 0;
    }
    const auto masked = [&](float v) { return kSigmoid ? !(v >= lowest) : !(v - largest >= kNothing); };
    // the softmax's sum
    float sum = 0;
    float inv = 0;
    if (!kSigmoid && (kBias || !c.renormalize)) {
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += exp_nonpositive(x.v[i][j] - largest);
      sum = lanes_sum<S::kLanes>(sum, lane);
      inv = sum > 0 ? 1 / sum : 0.0f;
    }
    // an FP32 score's error: a sigmoid's 2^-21; a softmax's that of its sum too (up to 22
    // additions in a row), and none is larger than 1 / sum
    const float error = kSigmoid ? 0x1p-21f : 0x1p-19f * inv;
    bool doubt = false;
    int mine;
    {
      int key[S::kSteps][4];
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i) {
        f4_t b{0, 0, 0, 0};
        if constexpr (kBias) b = *reinterpret_cast<const f4_t*>(bias + 4 * (S::kLanes * i + l));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = x.v[i][j];
          float k = v;
          bool out = masked(v);
          if constexpr (kBias) {
            k = (kSigmoid ? sigmoid_key(v) : exp_nonpositive(v - largest) * inv) + b[j];
            out |= !(k > minus_inf());  // (no short cut: a branch an expert would cost more)
          }
          key[i][j] = out ? kNone : ordered(k);
        }
      }
      mine = choose<S, kBias>(key, c, space, l, lane, error, doubt);
    }
    if constexpr (kBias) {
      doubt = doubt && !padding;
      if (__builtin_expect(__any(doubt), 0)) {
        double* keys = space.template row<double>(lane);
        double total = 0;
        const int64_t base = min(t, g.rows - 1) * g.stride;
        const auto exponential = [&](int e, float& v) {
          v = vq::load_act(g.logits, kDtype, base + e);
          const bool bad = kSigmoid ? v != v : !(v < __builtin_inff());
          if (bad) v = minus_inf();
          return exp(double(kSigmoid ? -v : v) - (kSigmoid ? 0.0 : double(largest)));
        };
        if constexpr (!kSigmoid) {
#pragma unroll 1
          for (int e = l; e < g.experts; e += S::kLanes) {
            float v;
            total += exponential(e, v);
          }
#pragma unroll
          for (int d = S::kLanes / 2; d > 0; d /= 2) total += __shfl_xor(total, d);
        }
        wave_lds_fence();
#pragma unroll 1
        for (int e = l; e < g.experts; e += S::kLanes) {
          float v;
          const double u = exponential(e, v);
          const double k = (kSigmoid ? 1 / (1 + u) : u / total) + double(bias[e]);
          keys[e] = masked(v) || !(k > -__builtin_inf()) ? -__builtin_inf() : k;
        }
        const int exact = choose_exact<S>(keys, c, g.experts, l);
        if (doubt) mine = exact;
      }
    }
    // slot l's weight in lane l
    const bool chosen = l < c.top_k && mine >= 0;
    const float v = chosen ? vq::load_act(g.logits, kDtype, min(t, g.rows - 1) * g.stride + mine) : minus_inf();
    float w = 0;
    if (c.renormalize) {
      // over the largest chosen one's size, so that shares do not depend on where logits lie
      float top = lanes_max<S::kLanes>(v, lane);
      if (top == minus_inf()) top = 0;
      if constexpr (kSigmoid) {
        const float k = top < 0 ? __builtin_ceilf(top * kLog2e) : 0.0f;
        const float u = exp_nonpositive(-fabsf(v));
        w = (v >= 0 ? 1.0f : exp_nonpositive(v, k)) / (1 + u);
      } else {
        w = exp_nonpositive(v - top);
      }
      w = chosen ? w : 0.0f;
      const float all = lanes_sum<S::kLanes>(w, lane);
      w = all > 0 ? w / all : 0.0f;
    } else if (chosen) {
      if constexpr (kSigmoid) {
        const float u = exp_nonpositive(-fabsf(v));
        w = (v >= 0 ? 1.0f : u) / (1 + u);
      } else {
        w = exp_nonpositive(v - largest) / sum;
      }
    }
    w *= c.scale;
    if (poisoned) w = chosen ? __builtin_nanf("") : 0.0f;
    if (t < g.rows && l < c.top_k) {
      c.weights[t * c.top_k + l] = padding || !chosen ? 0.0f : w;
      c.ids[t * c.top_k + l] = padding || !chosen ? -1 : mine;
    }
  }
}

struct Slots {
  const float* weights;
  const int32_t* ids;
  const float* upstream;
  int top_k;
  bool renormalize;
};

template <typename S, int kDtype, bool kSigmoid>
__global__ __launch_bounds__(kThreads) void grad_kernel(Rows g, Slots c, void* grad) {
  constexpr int kPadded = 4 * S::kLanes * S::kSteps;
  // the chosen experts' parts, zeros between the rows' turns
  __shared__ __attribute__((aligned(16))) float parts[kWaves][S::kRows * kPadded];
  typedef float f4_t __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, lane = tid & 63, wave = vq::uniform(tid >> 6);
  const int l = lane % S::kLanes, sub = lane / S::kLanes;
  float* part = parts[wave] + sub * kPadded;
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) *reinterpret_cast<f4_t*>(part + 4 * (S::kLanes * i + l)) = f4_t{0, 0, 0, 0};
  const bool wide = g.experts % 4 == 0;  // (rows of the gradient lie close)
  const bool dense = !kSigmoid && !c.renormalize;
  const int64_t step = int64_t(gridDim.x) * kWaves * S::kRows;
  for (int64_t t0 = (int64_t(blockIdx.x) * kWaves + wave) * S::kRows; t0 < g.rows; t0 += step) {
    const int64_t t = t0 + sub, at = min(t, g.rows - 1);
    int e = -1;
    float w = 0, up = 0;
    if (l < c.top_k) {
      e = c.ids[at * c.top_k + l];
      w = c.weights[at * c.top_k + l];
      up = c.upstream[at * c.top_k + l];
    }
    const bool chosen = e >= 0 && e < g.experts;
    if (!chosen) w = up = 0;
    float d = w * up, all = 0;
    if (c.renormalize) {
      // (shares of the weights' own sum: a single one's gradient is 0 as it stands)
      const float sum = lanes_sum<S::kLanes>(w, lane), share = sum != 0 ? w / sum : 0.0f;
      d = w * (up - lanes_sum<S::kLanes>(share * up, lane));
    } else if (!kSigmoid) {
      all = lanes_sum<S::kLanes>(d, lane);
    }
    if constexpr (kSigmoid) {
      // 1 - sigmoid of the logit is the sigmoid of its opposite
      const float v = chosen ? vq::load_act(g.logits, kDtype, at * g.stride + e) : 0.0f;
      d *= sigmoid_of(-v);
    }
    __builtin_amdgcn_wave_barrier();
    if (chosen) part[e] = d;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float out[S::kSteps][4];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      const f4_t p = *reinterpret_cast<const f4_t*>(part + 4 * (S::kLanes * i + l));
#pragma unroll
      for (int j = 0; j < 4; ++j) out[i][j] = p[j];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (chosen) part[e] = 0;
    if (dense) {
      const uint64_t any = __ballot(chosen);
      const bool used = (S::kLanes == 64 ? any : (any >> (S::kLanes * sub)) & ((uint64_t(1) << (S::kLanes & 63)) - 1)) != 0;
      const Values<S> x = load_row<S, kDtype>(g, at, l);
      float m = logits::row_max(x, lane), sum = 0;
      if (m == minus_inf()) m = 0;
      float z[S::kSteps][4];
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += z[i][j] = exp_nonpositive(x.v[i][j] - m);
      sum = lanes_sum<S::kLanes>(sum, lane);
      const float share = all / sum;
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) out[i][j] = used ? out[i][j] - z[i][j] * share : 0.0f;  // (rows that chose nothing may hold anything)
    }
    if (t >= g.rows) continue;
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      const int e0 = 4 * (S::kLanes * i + l);
      const int64_t to = t * g.experts + e0;
      if (wide && e0 < g.experts) {
        if constexpr (kDtype == vq::kFP32) {
          *reinterpret_cast<f4_t*>(static_cast<float*>(grad) + to) = f4_t{out[i][0], out[i][1], out[i][2], out[i][3]};
        } else {
          typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
          const auto half = [](float a) {
            return uint32_t(kDtype == vq::kBF16 ? vq::f32_to_bf16(a) : __builtin_bit_cast(uint16_t, _Float16(a)));
          };
          *reinterpret_cast<u2_t*>(static_cast<uint16_t*>(grad) + to) =
              u2_t{half(out[i][0]) | (half(out[i][1]) << 16), half(out[i][2]) | (half(out[i][3]) << 16)};
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (e0 + j < g.experts) vq::store_act(grad, kDtype, to + j, out[i][j]);
        }
      }
    }
  }
}

// launch(shape, dtype, sigmoid) for rows of `experts` whose lanes hold `slots` slots
// (and groups) at least.
template <typename F>
int dispatch(int64_t experts, int64_t slots, int dtype, bool sigmoid, const F& launch) {
  const auto shaped = [&](auto shape) {
    const auto typed = [&](auto type) {
      if (sigmoid) launch(shape, type, std::true_type{});
      else launch(shape, type, std::false_type{});
    };
    if (dtype == vq::kBF16) typed(std::integral_constant<int, vq::kBF16>{});
    else if (dtype == vq::kFP16) typed(std::integral_constant<int, vq::kFP16>{});
    else typed(std::integral_constant<int, vq::kFP32>{});
  };
  if (slots <= 16 && experts <= 64) shaped(Shape<16, 1>{});
  else if (slots <= 16 && experts <= 128) shaped(Shape<16, 2>{});
  else if (slots <= 16 && experts <= 256) shaped(Shape<16, 4>{});
  else if (experts <= 256) shaped(Shape<64, 1>{});
  else if (slots <= 32 && experts <= 512) shaped(Shape<32, 4>{});
  else shaped(Shape<64, 4>{});
  return vq::check_launch("moe_route_logits");
}

template <typename S>
unsigned grid_of(int64_t rows) {
  const int64_t each = kWaves * S::kRows;
  return unsigned(std::max<int64_t>(1, std::min<int64_t>(kMaxGrid, (rows + each - 1) / each)));
}

Rows rows_of(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const uint8_t* padding) {
  const int64_t four = 4 * vq::dtype_bytes(dtype);
  const bool wide = experts % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % four == 0;
  return {logits, stride, padding, rows, int(experts), wide};
}

int check_call(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, int64_t top_k, int scoring) {
  if (dtype != vq::kBF16 && dtype != vq::kFP16 && dtype != vq::kFP32) return vq::fail("moe_route_logits: logits must be BF16, FP16 or FP32");
  if (rows < 0 || rows > INT_MAX) return vq::fail("moe_route_logits: rows out of range");
  if (experts <= 0 || experts > kMaxExperts) return vq::fail("moe_route_logits: between 1 and 1024 experts");
  if (top_k <= 0 || top_k > kMaxSlots || top_k > experts) return vq::fail("moe_route_logits: topk must be between 1 and 64, and at most the experts");
  if (scoring != 0 && scoring != 1) return vq::fail("moe_route_logits: scoring must be softmax (0) or sigmoid (1)");
  if (stride < 0 || (rows > 1 && stride < experts) || stride > (int64_t(1) << 31)) return vq::fail("moe_route_logits: row stride out of range");
  if (rows > 0 && !logits) return vq::fail("moe_route_logits: null pointer");
  return vq::kOk;
}

// A call's arrays: no output may overlap another array, and each lies on its elements.
struct Span {
  const void* p;
  int64_t bytes, element;
};
int check_spans(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  for (const Span* a = outputs.begin(); a != outputs.end(); ++a) {
    for (const Span* b = outputs.begin(); b != a; ++b) {
      if (vq::overlaps(a->p, a->bytes, b->p, b->bytes)) return vq::fail("moe_route_logits: arguments must not overlap");
    }
    for (const Span& b : inputs) {
      if (vq::overlaps(a->p, a->bytes, b.p, b.bytes)) return vq::fail("moe_route_logits: arguments must not overlap");
    }
  }
  for (const auto* list : {&outputs, &inputs}) {
    for (const Span& a : *list) {
      if (reinterpret_cast<uintptr_t>(a.p) % uintptr_t(a.element)) return vq::fail("moe_route_logits: misaligned pointer");
    }
  }
  return vq::kOk;
}

int64_t logits_bytes(int dtype, int64_t rows, int64_t experts, int64_t stride) {
  return rows > 0 ? ((rows - 1) * stride + experts) * vq::dtype_bytes(dtype) : 0;
}

}  // namespace
}  // namespace route

extern "C" int moe_route_logits(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const float* bias,
                                int64_t top_k, int64_t groups, int64_t topk_groups, int scoring, int renormalize, float scale,
                                const uint8_t* is_padding, float* topk_weights, int32_t* topk_ids, void* stream) {
  using namespace route;
  if (int rc = check_call(logits, dtype, rows, experts, stride, top_k, scoring)) return rc;
  if (!(scale > -__builtin_inff() && scale < __builtin_inff())) return vq::fail("moe_route_logits: the scale must be finite");
  if (groups <= 0 || groups > kMaxGroups || experts % groups) return vq::fail("moe_route_logits: up to 64 groups of equal size");
  if (topk_groups <= 0 || topk_groups > groups) return vq::fail("moe_route_logits: topk_groups must be between 1 and the groups");
  if (top_k > topk_groups * (experts / groups)) return vq::fail("moe_route_logits: topk experts do not fit topk_groups groups");
  if (rows == 0) return vq::kOk;
  if (!topk_weights || !topk_ids) return vq::fail("moe_route_logits: null pointer");
  const int64_t slots = rows * top_k;
  if (int rc = check_spans({{topk_weights, slots * 4, 4}, {topk_ids, slots * 4, 4}},
                           {{logits, logits_bytes(dtype, rows, experts, stride), vq::dtype_bytes(dtype)},
                            {bias, experts * 4, 4}, {is_padding, rows, 1}})) {
    return rc;
  }
  if (topk_groups == groups) groups = topk_groups = 1;  // all are open
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Rows g = rows_of(logits, dtype, rows, experts, stride, is_padding);
  Choice c{bias, int(top_k), int(groups), int(topk_groups), int(experts / groups), 0, renormalize != 0, scale, topk_weights, topk_ids};
  return dispatch(experts, std::max(top_k, groups), dtype, scoring == 1, [&](auto shape, auto type, auto sigmoid) {
    using S = decltype(shape);
    const int lanes = c.group_experts / 4;
    if (c.group_experts % 4 == 0 && lanes <= S::kLanes && (lanes & (lanes - 1)) == 0) c.group_lanes = lanes;
    if (bias) {
      hipLaunchKernelGGL((choose_kernel<S, decltype(type)::value, decltype(sigmoid)::value, true>), dim3(grid_of<S>(rows)), dim3(kThreads), 0,
                         s, g, c);
    } else {
      hipLaunchKernelGGL((choose_kernel<S, decltype(type)::value, decltype(sigmoid)::value, false>), dim3(grid_of<S>(rows)), dim3(kThreads), 0,
                         s, g, c);
    }
  });
}

extern "C" int moe_route_grad(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t stride, const float* topk_weights,
                              const int32_t* topk_ids, int64_t top_k, int scoring, int renormalize, const float* upstream,
                              void* grad, void* stream) {
  using namespace route;
  if (int rc = check_call(logits, dtype, rows, experts, stride, top_k, scoring)) return rc;
  if (rows == 0) return vq::kOk;
  if (!topk_weights || !topk_ids || !upstream || !grad) return vq::fail("moe_route_logits: null pointer");
  const int64_t slots = rows * top_k, bytes = vq::dtype_bytes(dtype);
  if (int rc = check_spans({{grad, rows * experts * bytes, 4 * bytes}},
                           {{logits, logits_bytes(dtype, rows, experts, stride), bytes},
                            {topk_weights, slots * 4, 4}, {topk_ids, slots * 4, 4}, {upstream, slots * 4, 4}})) {
    return rc;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Rows g = rows_of(logits, dtype, rows, experts, stride, nullptr);
  const Slots c{topk_weights, topk_ids, upstream, int(top_k), renormalize != 0};
  return dispatch(experts, top_k, dtype, scoring == 1, [&](auto shape, auto type, auto sigmoid) {
    using S = decltype(shape);
    hipLaunchKernelGGL((grad_kernel<S, decltype(type)::value, decltype(sigmoid)::value>), dim3(grid_of<S>(rows)), dim3(kThreads), 0, s, g, c,
                       grad);
  });
}

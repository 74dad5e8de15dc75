// Routing of tokens to experts: scores, a balance bias, expert groups, top-k and the weights, one warp per token.
//
//   score_e  = softmax(logits)_e or sigmoid(logit_e)                         (0 for a masked expert, logit -inf)
//   choice_e = score_e + bias_e, or the logit itself without a bias          (same order as the score, and exact)
//   groups: a group's score is the sum of its best group_top live choices (with group_top = 2 and no bias: of its
//           best scores); the best top_groups groups stay
//   picks:  the top_k best choices of the experts that stay, equal choices by ascending index, masked experts last
//   weights: the picks' scores (without the bias), divided by their sum if asked for, times scale
//
// Which experts come out is decided as in 64 bits (what is equal there goes by ascending index): the fast form orders
// approximate choices that are off by less than half of a margin (below), and where two neighbouring picks, or the last
// group that stays and the first that goes, are closer than that, those picks (refine_picks) or groups (refine_groups)
// are compared again in 64 bits: about two rows in a thousand, and what a refinement takes is part of every larger call's
// time.  Equal inputs need no comparison, unless something else is near the place where the picks end.  Rows with a NaN,
// rows that have fewer live experts than picks and rows in which the candidates themselves are unsure (a finite mask of
// -1e9 on all of a lane's experts stretches the keys until everything else is near everything) are decided in 64 bits
// from the start (choose_exactly), at ten times the cost.
//
// Bound by instructions and their latency: at 65536 tokens x 256 experts the bytes take 11 us, and what a warp does per
// token decides.
//  * a lane holds VPL neighbouring experts, loaded with one or two vector loads; the bias stays in registers;
//  * the k best choices are no smaller than the smallest of the lanes' best ones (where more than k lanes have any):
//    that range, [lo, hi], is spread over 22 or 23 bits, which loses no more than fp32 does, and the expert's index,
//    counted down, takes the rest of a 32-bit key.  The largest key of the warp, one redux, then is the next pick with
//    its index, ties going to the lowest;
//  * a lane keeps its two best keys, and only a lane that has given up both looks through its experts again;
//  * the picks' logits are read again at the end, by lane r for pick r, instead of travelling through the rounds.
#include "common.cuh"

namespace hb200 {
namespace route {

constexpr int kWarps = 8;
constexpr unsigned kAll = 0xffffffffu;

struct Args {
  const void* logits;
  int64_t ld, tokens;
  const float* bias;  // [experts] or nullptr
  float* weights;
  int64_t* chosen;
  int experts, top_k, sigmoid, num_groups, top_groups, group_top, group_size, renormalize;
  int vec;            // a lane's experts can be read with vector loads
  int lanes_log;      // log2 of the lanes that look through a group
  int many_lanes_log; // the same where eight lanes hold a token
  uint32_t group_low; // 2^b - 1 >= num_groups - 1: the last b bits of a group score's key hold the group
  uint32_t group_inv; // ceil(2^20 / group_size): e / group_size = e * group_inv >> 20 for e < 1024
  float scale;
};

// Order-preserving keys: larger value, larger key; -0 counts as +0.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ float warp_max_of(float v) { return value_of(__reduce_max_sync(kAll, key_of(v))); }

template <typename R>
__device__ __forceinline__ R warp_total(R v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Accurate scores, for weights.
__device__ __forceinline__ float sigmoid_of(float v) {
  const float e = expf(-fabsf(v));
  return (v < 0.f ? e : 1.f) / (1.f + e);
}

// Scores for choices, from the hardware's exponential and reciprocal.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// softmax: exp(v - top) / total, otherwise the sigmoid
__device__ __forceinline__ float score_fast(float v, bool sigmoid, float top, float inv_total) {
  return sigmoid ? reciprocal_fast(1.f + exp2_fast(-kLog2e * v)) : exp2_fast(kLog2e * (v - top)) * inv_total;
}

template <typename T, int VPL>
__device__ __forceinline__ void load_row(const Args& a, const T* row, int lane, float (&l)[VPL]) {
  if (a.vec) {
    constexpr int kBytes = VPL * int(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
    __align__(16) T t[VPL];  // written in words of up to 16 bytes
    if (lane * VPL < a.experts) {
#pragma unroll
      for (int i = 0; i < kBytes / kWord; ++i) {
        const char* src = reinterpret_cast<const char*>(row + lane * VPL) + i * kWord;
        char* dst = reinterpret_cast<char*>(t) + i * kWord;
        if constexpr (kWord == 16) *reinterpret_cast<uint4*>(dst) = __ldg(reinterpret_cast<const uint4*>(src));
        else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(dst) = __ldg(reinterpret_cast<const uint2*>(src));
        else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(dst) = __ldg(reinterpret_cast<const uint32_t*>(src));
        else *reinterpret_cast<uint16_t*>(dst) = __ldg(reinterpret_cast<const uint16_t*>(src));
      }
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) l[j] = lane * VPL < a.experts ? float(t[j]) : -INFINITY;
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j) l[j] = lane * VPL + j < a.experts ? float(row[lane * VPL + j]) : -INFINITY;
  }
}

struct Picks {
  int expert;   // lane r holds pick r
  float logit;
};

// ------------------------------------------------------------------ 64-bit comparisons of what fp32 leaves unsure
// The softmax's sum, where an exact choice needs it (1 otherwise: it would scale both sides of a comparison).
template <typename T>
__device__ __forceinline__ double exact_total(const Args& a, const T* row, float top, int lane) {
  if (a.sigmoid || a.bias == nullptr) return 1.0;
  double total = 0.0;
  for (int e = lane; e < a.experts; e += 32) {
    const float l = float(row[e]);
    if (l > -INFINITY) total += exp(double(l) - double(top));
  }
  return warp_total(total);
}

// Score (of_score) or logit, plus the bias.
__device__ __forceinline__ double exact_choice(const Args& a, float logit, int e, float top, double total, bool of_score) {
  double c = double(logit);
  if (of_score) {
    const double t = a.sigmoid ? exp(-fabs(c)) : exp(c - double(top));
    c = a.sigmoid ? (c < 0.0 ? t : 1.0) / (1.0 + t) : t / total;
  }
  return a.bias != nullptr ? c + double(a.bias[e]) : c;
}

// Whether the group of this lane stays.  `sure`: its score lies clear above every group that would go; `near`: it does
// not, nor clear below every group that would stay, and is compared by its exact score.
template <typename T>
__device__ __noinline__ bool refine_groups(const Args& a, const T* row, float top, int group, bool sure, bool near) {
  const int lane = threadIdx.x & 31, lanes = 1 << a.lanes_log;
  const bool of_score = a.bias != nullptr || a.group_top > 1;
  const double total = exact_total(a, row, top, lane);
  const unsigned near_lanes = __ballot_sync(kAll, near);
  const int sure_groups = __popc(__ballot_sync(kAll, sure && (lane & (lanes - 1)) == 0));
  double mine = -INFINITY;
  for (int g = 0; g < a.num_groups; ++g) {
    if (!((near_lanes >> (g << a.lanes_log)) & 1u)) continue;
    double b1 = -INFINITY, b2 = -INFINITY;
    for (int i = lane; i < a.group_size; i += 32) {
      const int e = g * a.group_size + i;
      const float l = float(row[e]);
      if (!(l > -INFINITY)) continue;
      const double c = exact_choice(a, l, e, top, total, of_score);
      if (c > b1) b2 = b1, b1 = c; else if (c > b2) b2 = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
      const double low = o1 < b1 ? o1 : b1, high = o1 < b1 ? b1 : o1, second = o2 < b2 ? b2 : o2;
      b1 = high;
      b2 = low > second ? low : second;
    }
    if (group == g) mine = a.group_top > 1 && b2 > -INFINITY ? b1 + b2 : b1;
  }
  int before = 0;
  for (int g = 0; g < a.num_groups; ++g) {
    const double other = __shfl_sync(kAll, mine, g << a.lanes_log);
    if ((near_lanes >> (g << a.lanes_log)) & 1u) before += other > mine || (other == mine && g < group);
  }
  return sure || (near && before < a.top_groups - sure_groups);
}

// The picks of lanes 0 .. count - 1 in the order of their exact choices.
template <typename T>
__device__ __noinline__ Picks refine_picks(const Args& a, const T* row, float top, Picks p, int count) {
  const int lane = threadIdx.x & 31;
  const bool has = lane < count;
  const double total = exact_total(a, row, top, lane);
  const double mine = has ? exact_choice(a, p.logit, p.expert, top, total, a.bias != nullptr) : 0.0;
  int rank = 0;
  for (int r = 0; r < count; ++r) {
    const double other = __shfl_sync(kAll, mine, r);
    const int expert = __shfl_sync(kAll, p.expert, r);
    rank += other > mine || (other == mine && expert < p.expert);
  }
  int from = lane;
  for (int r = 0; r < count; ++r)
    if (__shfl_sync(kAll, rank, r) == lane) from = r;
  return Picks{__shfl_sync(kAll, p.expert, from), __shfl_sync(kAll, p.logit, from)};
}

// ------------------------------------------------------------------ exact form, for the few rows that need it
__device__ __forceinline__ double warp_best(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double other = __shfl_xor_sync(kAll, v, o);
    v = other > v ? other : v;
  }
  return v;
}

template <typename T, int VPL>
__device__ __noinline__ Picks choose_exactly(const Args& a, const T* row, int lane) {
  float l[VPL];
  load_row<T, VPL>(a, row, lane, l);
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < VPL; ++j) top = fmaxf(top, l[j]);
  top = warp_max_of(top);
  double total = 0.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (l[j] > -INFINITY) total += exp(double(l[j]) - double(top));
    total = warp_total(total);
  }
  auto score = [&](double v) {
    if (!a.sigmoid) return exp(v - double(top)) / total;
    const double e = exp(v < 0.0 ? v : -v);
    return (v < 0.0 ? e : 1.0) / (1.0 + e);
  };
  // rank: 2 live, 1 masked, 0 not to be picked (any more); within a rank the choice decides (masked: the index alone)
  double choice[VPL];
  uint32_t live = 0, open = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = lane * VPL + j;
    choice[j] = double(l[j]);
    if (a.bias != nullptr && e < a.experts && l[j] > -INFINITY) choice[j] = score(double(l[j])) + double(a.bias[e]);
    if (e < a.experts) open |= 1u << j;
    if (e < a.experts && l[j] > -INFINITY && choice[j] > -INFINITY) live |= 1u << j;
  }
  if (a.num_groups > 1) {
    const bool of_scores = a.group_top > 1 && a.bias == nullptr;
    double mine = -INFINITY;
    for (int g = 0; g < a.num_groups; ++g) {
      const int lo = g * a.group_size, hi = lo + a.group_size;
      double s = -INFINITY;
      uint32_t left = live;
      for (int i = 0; i < a.group_top; ++i) {
        double m = -INFINITY;
        int at_j = -1;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          const int e = lane * VPL + j;
          if (e >= lo && e < hi && ((left >> j) & 1u) && (at_j < 0 || choice[j] > m)) m = choice[j], at_j = j;
        }
        const unsigned some = __ballot_sync(kAll, at_j >= 0);
        if (some == 0) break;
        const double best = warp_best(m);
        const int at = __ffs(__ballot_sync(kAll, at_j >= 0 && m == best)) - 1;
        if (lane == at) left &= ~(1u << at_j);
        const double value = of_scores ? score(best) : best;
        s = i == 0 ? value : s + value;
      }
      if (lane == g) mine = s;
    }
    int before = 0;
    for (int g = 0; g < a.num_groups; ++g) {
      const double other = __shfl_sync(kAll, mine, g);
      before += other > mine || (other == mine && g < lane);
    }
    const unsigned kept = __ballot_sync(kAll, lane < a.num_groups && before < a.top_groups);
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if ((open >> j) & 1u && !((kept >> ((lane * VPL + j) / a.group_size)) & 1u)) open &= ~(1u << j);
  }
  Picks p{0, -INFINITY};
  for (int r = 0; r < a.top_k; ++r) {
    int rank = 0, at_j = 0;
    double m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      if (!((open >> j) & 1u)) continue;
      const int mine = 1 + int((live >> j) & 1u);
      if (mine > rank || (mine == rank && mine == 2 && choice[j] > m)) rank = mine, m = choice[j], at_j = j;
    }
    const int best_rank = __reduce_max_sync(kAll, rank);
    const double best = warp_best(rank == best_rank && rank == 2 ? m : -INFINITY);
    const int at = __ffs(__ballot_sync(kAll, rank == best_rank && (rank < 2 || m == best))) - 1;
    float logit = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (j == at_j) logit = l[j];
    if (lane == at) open &= ~(1u << at_j);
    const int e = __shfl_sync(kAll, lane * VPL + at_j, at);
    logit = __shfl_sync(kAll, logit, at);
    if (lane == r) p.expert = e, p.logit = logit;
  }
  return p;
}

// ------------------------------------------------------------------ fast form
constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN wins
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float redux_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float redux_min(float v) {
  float r;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// What two choices may be off by, together.  Sigmoid: 14 units of 2^-24 (its argument's rounding, one exponential, one
// addition, one reciprocal, of values up to 1, twice); softmax: up to 60 (the rounding of logit - top scaled by the
// score, the sum's own error, twice); additions half a unit in the last place each come on top.  Without a bias the
// logits themselves are compared.
__device__ __forceinline__ float choice_error(const Args& a) {
  return a.bias == nullptr ? 0.f : (a.sigmoid ? 1.f / (1 << 20) : 1.f / (1 << 18));
}

// What a group's score s may be off by: `error` for its one or two choices, the rounding of each of these (m1 and, where
// m2 is above -infinity, m2: a sum can be far smaller than they are; 0 where none was rounded) and of their sum, and what
// the group's place takes of the key.
__device__ __forceinline__ float group_error(float s, float m1, float m2, float error, uint32_t group_low) {
  const float larger = fmaxf(fabsf(m1), m2 > -INFINITY ? fabsf(m2) : 0.f);
  const float off = error + larger * (1.f / (1 << 23)) + fabsf(s) * (float(group_low + 2) * (1.f / (1 << 23))) + 1e-36f;
  return fabsf(s) < INFINITY ? off : 0.f;
}

// How groups lie in the lanes: none, whole lanes (a power of two of them) per group, or anyhow.
enum Groups { kNoGroups = 0, kLaneGroups = 1, kAnyGroups = 2 };

// Weights of a token's picks (lane r holds pick r), and the result.  Renormalised weights are ratios of scores: they are
// formed relative to the largest pick, so that picks far below the row's largest logit (a bias or a group can choose
// them) keep their ratios.
__device__ __forceinline__ void write_weights(const Args& a, int64_t token, const Picks& p, float top, float total, bool spoilt) {
  const int lane = threadIdx.x & 31;
  const bool sigmoid = a.sigmoid != 0, has_pick = lane < a.top_k, live = has_pick && p.logit > -INFINITY;
  float w = 0.f;
  if (a.renormalize) {
    const float best = redux_max_nan(live ? p.logit : -INFINITY);
    if (!sigmoid) {
      w = live ? expf(p.logit - best) : 0.f;
    } else {
      // relative to the best pick's exp(best) where that is negative
      const float t = expf(-fabsf(p.logit));
      float numerator = p.logit < 0.f ? t : 1.f;
      if (best < 0.f) numerator = expf(p.logit - best);
      w = live ? __fdividef(numerator, 1.f + t) : 0.f;
    }
    const float sum = warp_total(w);
    if (live) w = __fdividef(w, sum);
  } else if (live) {
    w = sigmoid ? sigmoid_of(p.logit) : __fdividef(expf(p.logit - top), total);
  }
  w = spoilt ? NAN : w * a.scale;
  if (has_pick) {
    a.weights[token * a.top_k + lane] = w;
    a.chosen[token * a.top_k + lane] = p.expert;
  }
}

// One token, a warp.  b: the lane's biases (0 without one).
template <typename T, int VPL, int GROUPS>
__device__ __forceinline__ void route_token(const Args& a, int64_t token, const float (&b)[VPL], float* my_choices) {
  constexpr int kIndexBits = 5 + log2_of(VPL), kValueBits = kIndexBits <= 9 ? 23 : 32 - kIndexBits;
  constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
  const int lane = threadIdx.x & 31;
  const bool sigmoid = a.sigmoid != 0, biased = a.bias != nullptr;
  const bool by_scores = GROUPS != kNoGroups && a.group_top > 1;  // group scores are sums of scores
  const float base = choice_error(a);
  const T* row = static_cast<const T*>(a.logits) + token * a.ld;
  float c[VPL];  // logits, then choices
  load_row<T, VPL>(a, row, lane, c);
  float top = 0.f, total = 0.f, inv_total = 0.f;
  float hi = c[0];  // a lane's best choice
#pragma unroll
  for (int j = 1; j < VPL; ++j) hi = max_nan(hi, c[j]);
  // A NaN (or, under softmax, an infinite logit) spoils the row's scores: its weights come out as NaN.
  bool spoilt = false;
  if (!sigmoid) {
    top = redux_max_nan(hi);
    spoilt = top == INFINITY;
    if (biased || by_scores || !a.renormalize) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) total += exp2_fast(kLog2e * (c[j] - top));
      total = warp_total(total);
      inv_total = reciprocal_fast(total);
    }
  }
  if (biased) {
    float low = c[0];
#pragma unroll
    for (int j = 1; j < VPL; ++j) low = fminf(low, c[j]);
    float choice[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) choice[j] = score_fast(c[j], sigmoid, top, inv_total) + b[j];
    if (low == -INFINITY) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) choice[j] = c[j] == -INFINITY ? -INFINITY : choice[j];
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) c[j] = choice[j], hi = j == 0 ? c[0] : max_nan(hi, c[j]);
  }
  spoilt = __any_sync(kAll, spoilt || hi != hi);
  bool slow = spoilt;  // decided by choose_exactly

  bool alive = hi > -INFINITY;  // this lane has experts to pick
  if constexpr (GROUPS != kNoGroups) {
    // the two best choices of the group that this lane looks through: its own experts' group, or (any layout) one
    // that 2^lanes_log lanes share
    const int lanes = 1 << a.lanes_log, group = lane >> a.lanes_log;
    const bool is_group = group < a.num_groups;
    float m1 = -INFINITY, m2 = -INFINITY;
    if constexpr (GROUPS == kLaneGroups) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) m2 = fmaxf(m2, fminf(m1, c[j])), m1 = fmaxf(m1, c[j]);
    } else {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < VPL; ++j) my_choices[lane * VPL + j] = c[j];
      __syncwarp();
      if (is_group) {
        for (int i = lane & (lanes - 1); i < a.group_size; i += lanes) {
          const float v = my_choices[group * a.group_size + i];
          m2 = fmaxf(m2, fminf(m1, v));
          m1 = fmaxf(m1, v);
        }
      }
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const float o1 = __shfl_xor_sync(kAll, m1, o), o2 = __shfl_xor_sync(kAll, m2, o);
      m2 = fmaxf(fmaxf(m2, o2), fminf(m1, o1));
      m1 = fmaxf(m1, o1);
    }
    const bool convert = by_scores && !biased;
    float s = m1;
    if (convert && m1 > -INFINITY) s = score_fast(m1, sigmoid, top, inv_total);
    if (by_scores && m2 > -INFINITY) s += convert ? score_fast(m2, sigmoid, top, inv_total) : m2;
    // a group's rank: its score's key with the group, counted down, in the last bits
    const uint32_t s_key = is_group ? (key_of(s) & ~a.group_low) | (a.group_low - uint32_t(group)) : 0u;
    int before = 0;
#pragma unroll 4
    for (int g = 0; g < a.num_groups; ++g) before += __shfl_sync(kAll, s_key, g << a.lanes_log) > s_key;
    bool stays = is_group && before < a.top_groups;
    const float error = base + (convert ? 1.f / (1 << 18) : 0.f);
    if (a.top_groups < a.num_groups && !(error == 0.f && sizeof(T) == 2)) {  // (16-bit logits lose nothing to the keys)
      const float off = group_error(s, biased ? m1 : 0.f, biased && by_scores ? m2 : 0.f, error, a.group_low);
      const float last = redux_min(stays ? s - off : INFINITY), next = redux_max_nan(is_group && !stays ? s + off : -INFINITY);
      if (next > -INFINITY && last <= next && !spoilt) {
        const bool sure = stays && s - off > next;
        stays = refine_groups<T>(a, row, top, group, sure, is_group && !sure && s + off >= last);
      }
    }
    if constexpr (GROUPS == kLaneGroups) {
      alive = alive && stays;
      if (!alive) hi = -INFINITY;
    } else {
      const unsigned kept = __ballot_sync(kAll, stays);
      hi = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const uint32_t g = (uint32_t(lane * VPL + j) * a.group_inv) >> 20;
        if (!((kept >> ((g << a.lanes_log) & 31u)) & 1u)) c[j] = -INFINITY;
        hi = max_nan(hi, c[j]);
      }
      alive = hi > -INFINITY;
    }
  }

  // [lo, hi]: what the picks lie in
  float lo = redux_min(alive ? hi : INFINITY);
  hi = redux_max_nan(hi);
  if (__popc(__ballot_sync(kAll, alive)) <= a.top_k) {  // too few lanes: the smallest live choice bounds the picks
    lo = INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) lo = c[j] > -INFINITY ? fminf(lo, c[j]) : lo;
    lo = redux_min(alive ? lo : INFINITY);
  }
  const float range = hi - lo, largest = fmaxf(fabsf(hi), fabsf(lo));
  slow |= !(largest < 1e30f);  // infinite, or so large that a group's sum may have left fp32
  const float scale = float((1 << kValueBits) - 600) * reciprocal_fast(fmaxf(range, 1e-30f));
  // value 0: below lo, masked or dropped; 1 and up: in the range.  Added to 2^23 it is the sum's last 23 bits, and
  // what 2^23 itself would leave in the key goes with the index's constant.
  uint32_t key[VPL], m1 = 0, m2 = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const float q = fmaxf(fmaf(c[j] - lo, scale, 8388609.f), 8388608.f);
    key[j] = (__float_as_uint(q) << kIndexBits) + (kIndexMask - uint32_t(lane * VPL + j) - (0x4b000000u << kIndexBits));
    m2 = max(m2, min(m1, key[j]));
    m1 = max(m1, key[j]);
  }
  if (!alive) m1 = 0;
  uint32_t pick = 0, left = 0;
  for (int r = 0; r <= a.top_k; ++r) {  // one more, to compare the last pick with what it left behind
    left = __reduce_max_sync(kAll, m1);
    if (lane == r) pick = left;
    const bool mine = m1 == left;
    m1 = mine ? m2 : m1;
    m2 = mine ? 0 : m2;
    if (mine && m1 == 0) {  // both given up
#pragma unroll
      for (int j = 0; j < VPL; ++j) m1 = key[j] < left ? max(m1, key[j]) : m1;
    }
  }

  const bool has_pick = lane < a.top_k;
  slow = __any_sync(kAll, slow || (has_pick && (pick >> kIndexBits) == 0));
  Picks p{int(kIndexMask - (pick & kIndexMask)), -INFINITY};
  if (!slow) {
    if (has_pick) p.logit = float(row[p.expert]);
    uint32_t next = __shfl_down_sync(kAll, pick, 1);
    if (lane == a.top_k - 1) next = left;
    // in units of the keys' values: the choices' error, and two for the values' own rounding
    const float margin = fmaf(scale, base + largest * (1.f / (1 << 22)), 2.f);
    const bool near = has_pick && (next >> kIndexBits) != 0 && float((pick >> kIndexBits) - (next >> kIndexBits)) <= margin;
    const unsigned near_picks = __ballot_sync(kAll, near);
    if (near_picks != 0) {
      auto bias_of = [&](int e) { return biased ? a.bias[e] : 0.f; };
      bool unlike = near;
      if (near) {  // equal inputs are a tie whatever the precision, and in their order already
        const int e = int(kIndexMask - (next & kIndexMask));
        unlike = !(p.logit == float(row[e]) && bias_of(p.expert) == bias_of(e));
      }
      const bool some = __any_sync(kAll, unlike);
      int count = a.top_k;
      if ((near_picks >> (a.top_k - 1)) & 1u) {
        // The last pick and the expert left behind are near each other, equal or not: what follows that one within the
        // margin may come before both.  Only where all of these have the same inputs is it known which of them is picked.
        const int e_left = int(kIndexMask - (left & kIndexMask));
        const float l_left = float(row[e_left]), b_left = bias_of(e_left);
        bool more = false, other = false;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          // (value 0 lies below lo, by how little is not known: it counts as lo itself)
          const int e = lane * VPL + j;
          if (alive && e < a.experts && key[j] < left && float((left >> kIndexBits) - max(key[j] >> kIndexBits, 1u)) <= margin) {
            const float l = float(row[e]);
            if (l > -INFINITY) more = true, other |= !(l == l_left && bias_of(e) == b_left);
          }
        }
        count = a.top_k + 1;  // the one left behind takes part
        slow = __any_sync(kAll, some ? more || count > 32 : other);
        if (lane == a.top_k) p.expert = e_left, p.logit = l_left;
      }
      if (some && !slow) p = refine_picks<T>(a, row, top, p, count);
    }
  }
  if (slow) p = choose_exactly<T, VPL>(a, row, lane);

  write_weights(a, token, p, top, total, spoilt);
}

template <int VPL>
__device__ __forceinline__ void load_bias(const Args& a, float (&b)[VPL]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < VPL; ++j) b[j] = (a.bias != nullptr && lane * VPL + j < a.experts) ? a.bias[lane * VPL + j] : 0.f;
}

// CTAs per SM (the exact form, a call that few rows make, would otherwise set the registers and with them the occupancy);
// the grid is that many and every warp takes its tokens in turn, so all of them end within a token of each other.
template <int VPL> constexpr int kResident = VPL <= 8 ? 4 : (VPL == 16 ? 2 : 1);

template <typename T, int VPL, int GROUPS>
__global__ void __launch_bounds__(kWarps * 32, kResident<VPL>)
route_experts_kernel(const __grid_constant__ Args a) {
  __shared__ float shared_choices[GROUPS == kAnyGroups ? kWarps : 1][GROUPS == kAnyGroups ? 32 * VPL : 1];
  float b[VPL];
  load_bias<VPL>(a, b);
  const int64_t step = int64_t(gridDim.x) * kWarps;
  for (int64_t token = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); token < a.tokens; token += step)
    route_token<T, VPL, GROUPS>(a, token, b, shared_choices[GROUPS == kAnyGroups ? threadIdx.x >> 5 : 0]);
}

// ------------------------------------------------------------------ many tokens
// Four tokens per warp, eight lanes each: what a warp does once per round, group and row then serves four tokens.  A
// lane holds up to 32 neighbouring experts (staged through shared memory, so that the loads are coalesced and the next
// tokens' rows are on their way meanwhile) and keeps its four best keys.  The range of the keys starts at the smallest
// of the lanes' second-best choices where that leaves enough experts in it.  Tokens with near ties among their picks have
// these compared in 64 bits afterwards, by the whole warp; a token with anything else unsure goes through route_token.
// 65536 tokens x 256 experts, top 8: 46 us in groups (top 4 of 8, biased sigmoid) against 63 with a warp per token, 32
// against 39 by softmax; 128 experts in bf16 22 against 35, 64 in fp32 16 against 29.  410 instructions per token, issue
// slots busy 59 % at 14 warps per SM (128 registers): instructions and their latency share the time.  In smaller batches
// the longer work per warp shows as latency, hence the bounds in launch_many.  Here / a warp per token, fp32, top 6:
//   by softmax    4096 tokens   8192        16384       groups        8192        16384       32768
//   32 experts    3.2 / 2.8     5.1 / 4.1   6.2 / 6.5
//   64            3.6 / 3.5     4.4 / 5.6   6.6 / 8.4                 7.2 / 7.9   9.2 / 13.1  18.1 / 24.9
//   96            4.0 / 4.0     5.0 / 6.0   7.6 / 9.1
//   128           4.0 / 4.0     6.2 / 6.0   9.0 / 9.1                 12.7 / 10.3 16.6 / 14.3 20.9 / 27.8
//   192           4.6 / 5.0     7.2 / 7.3   10.3 / 10.8               8.8 / 13.6  18.4 / 21.1 25.2 / 37.4
//   256           4.5 / 4.9     6.2 / 7.3   10.1 / 10.7               13.4 / 12.2 18.8 / 18.1 25.6 / 31.4
constexpr int kManyWarps = 4;
constexpr int kManyMaxPicks = 8;

__device__ __forceinline__ float eight_max_nan(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = max_nan(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ float eight_min(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = fminf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ float eight_sum(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ uint32_t eight_max(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

template <typename T, int GROUPS>
__device__ __noinline__ void route_token_apart(const Args& a, int64_t token, float* scratch) {
  float b[8];
  load_bias<8>(a, b);
  route_token<T, 8, GROUPS>(a, token, b, scratch);
}

template <typename T>
__device__ __noinline__ void refine_apart(const Args& a, int64_t token, float top, float total, Picks p, int count) {
  p = refine_picks<T>(a, static_cast<const T*>(a.logits) + token * a.ld, top, p, count);
  write_weights(a, token, p, top, total, false);
}

template <typename T, int VPL, bool GROUPED>
__global__ void __launch_bounds__(kManyWarps * 32, VPL <= 16 ? 6 : 4)
route_many_kernel(const __grid_constant__ Args a) {
  constexpr int kLaneBytes = VPL * int(sizeof(T)) + 16;  // the pad spreads eight lanes' 16-byte reads over the banks
  constexpr int kRowBytes = 8 * kLaneBytes, kChunks = VPL * int(sizeof(T)) / 16;  // 16-byte chunks of a lane
  constexpr int kIndexBits = VPL <= 16 ? 7 : 8, kValueBits = 23;
  constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;
  __shared__ __align__(16) uint8_t staged[kManyWarps][2][4 * kRowBytes];
  __shared__ __align__(16) float shared_bias[8 * (VPL + 4)];
  __shared__ float scratch[GROUPED ? kManyWarps : 1][GROUPED ? 256 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane >> 3, l8 = lane & 7;
  const bool sigmoid = a.sigmoid != 0, biased = a.bias != nullptr, by_scores = GROUPED && a.group_top > 1;
  const float base = choice_error(a);
  for (int e = threadIdx.x; e < 8 * VPL; e += kManyWarps * 32)
    shared_bias[e / VPL * (VPL + 4) + e % VPL] = (biased && e < a.experts) ? a.bias[e] : 0.f;
  __syncthreads();

  const int chunks = a.experts * int(sizeof(T)) / 16;  // of a row
  auto fetch = [&](int64_t first, int buf) {
    const int64_t token = first + part < a.tokens ? first + part : a.tokens - 1;
    const uint8_t* src = static_cast<const uint8_t*>(a.logits) + token * a.ld * int64_t(sizeof(T));
    uint8_t* dst = staged[warp][buf] + part * kRowBytes;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int q = i * 8 + l8;
      if (q < chunks)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                     ::"r"(uint32_t(__cvta_generic_to_shared(dst + q / kChunks * kLaneBytes + q % kChunks * 16))),
                     "l"(src + q * 16)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  const int64_t step = int64_t(gridDim.x) * kManyWarps * 4;
  int64_t first = (int64_t(blockIdx.x) * kManyWarps + warp) * 4;
  int buf = 0;
  if (first < a.tokens) fetch(first, 0);
  for (; first < a.tokens; first += step, buf ^= 1) {
    if (first + step < a.tokens) fetch(first + step, buf ^ 1);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint8_t* rows = staged[warp][buf] + part * kRowBytes;
    const int64_t token = first + part;
    bool unsure = false;  // goes through route_token

    float c[VPL];  // logits, then choices
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(rows + l8 * kLaneBytes + i * 16);
      const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < 16 / int(sizeof(T)); ++j) c[i * (16 / int(sizeof(T))) + j] = float(t[j]);
    }
    if ((l8 + 1) * VPL > a.experts) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) c[j] = l8 * VPL + j < a.experts ? c[j] : -INFINITY;
    }
    float top = 0.f, total = 0.f, inv_total = 0.f;
    if (!sigmoid) {
      top = c[0];
#pragma unroll
      for (int j = 1; j < VPL; ++j) top = max_nan(top, c[j]);
      top = eight_max_nan(top);
      if (biased || by_scores || !a.renormalize) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) total += exp2_fast(kLog2e * (c[j] - top));
        total = eight_sum(total);
        inv_total = reciprocal_fast(total);
      }
      unsure = !(top > -INFINITY && top < INFINITY);
    }
    if (biased) {
      float low = c[0];
#pragma unroll
      for (int j = 1; j < VPL; ++j) low = fminf(low, c[j]);
      const float4* bias = reinterpret_cast<const float4*>(shared_bias + l8 * (VPL + 4));
      if (low == -INFINITY) {
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          c[j] = c[j] == -INFINITY ? -INFINITY : score_fast(c[j], sigmoid, top, inv_total) + reinterpret_cast<const float*>(bias)[j];
      } else {
#pragma unroll
        for (int j = 0; j < VPL / 4; ++j) {
          const float4 v = bias[j];
          c[4 * j] = score_fast(c[4 * j], sigmoid, top, inv_total) + v.x;
          c[4 * j + 1] = score_fast(c[4 * j + 1], sigmoid, top, inv_total) + v.y;
          c[4 * j + 2] = score_fast(c[4 * j + 2], sigmoid, top, inv_total) + v.z;
          c[4 * j + 3] = score_fast(c[4 * j + 3], sigmoid, top, inv_total) + v.w;
        }
      }
    }
    // the lane's two best choices (a NaN takes the first place)
    float hi = c[0], second = -INFINITY;
#pragma unroll
    for (int j = 1; j < VPL; ++j) second = fmaxf(second, fminf(hi, c[j])), hi = max_nan(hi, c[j]);
    const float best = eight_max_nan(hi);
    unsure |= !(best < INFINITY);  // a NaN, an infinite choice
    bool alive = hi > -INFINITY;
    if constexpr (GROUPED) {
      const int lanes = 1 << a.many_lanes_log, group = l8 >> a.many_lanes_log;
      const bool is_group = group < a.num_groups;
      float m1 = hi, m2 = second;
      for (int o = 1; o < lanes; o <<= 1) {
        const float o1 = __shfl_xor_sync(kAll, m1, o), o2 = __shfl_xor_sync(kAll, m2, o);
        m2 = fmaxf(fmaxf(m2, o2), fminf(m1, o1));
        m1 = fmaxf(m1, o1);
      }
      const bool convert = by_scores && !biased;
      float s = m1;
      if (convert && m1 > -INFINITY) s = score_fast(m1, sigmoid, top, inv_total);
      if (by_scores && m2 > -INFINITY) s += convert ? score_fast(m2, sigmoid, top, inv_total) : m2;
      const uint32_t s_key = is_group ? (key_of(s) & ~7u) | uint32_t(7 - group) : 0u;
      int before = 0;
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (g < a.num_groups) before += __shfl_sync(kAll, s_key, (lane & 24) + (g << a.many_lanes_log)) > s_key;
      const bool stays = is_group && before < a.top_groups;
      const float error = base + (convert ? 1.f / (1 << 18) : 0.f);
      if (a.top_groups < a.num_groups && !(error == 0.f && sizeof(T) == 2)) {
        const float off = group_error(s, biased ? m1 : 0.f, biased && by_scores ? m2 : 0.f, error, 7);
        const float last = eight_min(stays ? s - off : INFINITY), next = eight_max_nan(is_group && !stays ? s + off : -INFINITY);
        unsure |= next > -INFINITY && last <= next;
      }
      alive = alive && stays;
    }

    // [lo, hi]: the lanes' second-best choices leave two experts per live lane in it
    float lo = eight_min(alive ? second : INFINITY);
    const int lanes_alive = __popc((__ballot_sync(kAll, alive) >> (lane & 24)) & 255u);
    if (2 * lanes_alive < a.top_k || !(lo > -INFINITY)) {
      lo = INFINITY;
#pragma unroll
      for (int j = 0; j < VPL; ++j) lo = c[j] > -INFINITY ? fminf(lo, c[j]) : lo;
      if (!alive) lo = INFINITY;
    }
    lo = eight_min(lo);
    hi = eight_max_nan(alive ? hi : -INFINITY);
    lo -= 0.125f * (hi - lo);  // room below, so that what is left behind is not mistaken for a neighbour of the last pick
    const float range = hi - lo, largest = fmaxf(fabsf(hi), fabsf(lo));
    unsure |= !(largest < 1e30f);
    const float scale = float((1 << kValueBits) - 600) * reciprocal_fast(fmaxf(range, 1e-30f));
    uint32_t key[VPL], m1 = 0, m2 = 0, m3 = 0, m4 = 0;
    const uint32_t index = kIndexMask - uint32_t(l8 * VPL) - (0x4b000000u << kIndexBits);
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const float q = fmaxf(fmaf(c[j] - lo, scale, 8388609.f), 8388608.f);
      key[j] = (__float_as_uint(q) << kIndexBits) + (index - uint32_t(j));
      m4 = max(m4, min(m3, key[j]));
      m3 = max(m3, min(m2, key[j]));
      m2 = max(m2, min(m1, key[j]));
      m1 = max(m1, key[j]);
    }
    if (!alive) m1 = m2 = m3 = m4 = 0;
    uint32_t pick = 0, left = 0;
    for (int r = 0; r <= a.top_k; ++r) {
      left = eight_max(m1);
      if (l8 == r) pick = left;
      const bool mine = m1 == left && left != 0;
      if (mine) m1 = m2, m2 = m3, m3 = m4, m4 = 0;
      if (mine && m1 == 0) {  // all four given up
#pragma unroll
        for (int j = 0; j < VPL; ++j) m1 = key[j] < left ? max(m1, key[j]) : m1;
      }
    }

    const bool has_pick = l8 < a.top_k;
    uint32_t next = __shfl_down_sync(kAll, pick, 1);
    if (l8 == a.top_k - 1) next = left;
    const uint32_t value = pick >> kIndexBits, next_value = next >> kIndexBits;
    const int expert = min(int(kIndexMask - (pick & kIndexMask)), a.experts - 1);
    auto logit_of = [&](int e) {
      return float(*reinterpret_cast<const T*>(rows + e / VPL * kLaneBytes + e % VPL * int(sizeof(T))));
    };
    const float logit = has_pick ? logit_of(expert) : -INFINITY;
    // one more than in route_token: what was left behind may lie below lo
    const float margin = fmaf(scale, base + largest * (1.f / (1 << 22)), 3.f);
    const bool near = has_pick && next != 0 && float(value - next_value) <= margin;
    bool close = near;
    if (__any_sync(kAll, close)) {
      if (close) {  // equal inputs are a tie whatever the precision, and in their order already
        const int e = min(int(kIndexMask - (next & kIndexMask)), a.experts - 1);
        close = !(next_value != 0 && logit == logit_of(e) && (!biased || a.bias[expert] == a.bias[e]));
      }
    }
    unsure |= has_pick && value == 0;
    const unsigned close_lanes = __ballot_sync(kAll, close), edge_lanes = __ballot_sync(kAll, near && l8 == a.top_k - 1);
    if (edge_lanes != 0) {
      // The last pick and the expert left behind are near each other, equal or not: what follows that one within the
      // margin may come before both.  Only where all of these have the same inputs is it known which of them is picked.
      const uint32_t beyond = eight_max(m1), left_value = left >> kIndexBits;
      const bool deep = ((edge_lanes >> (lane & 24)) & 255u) != 0 &&
                        !(left_value != 0 && float(left_value - (beyond >> kIndexBits)) > margin);
      if (__any_sync(kAll, deep)) {
        bool other = false;
        if (deep && alive) {
          const int e_left = min(int(kIndexMask - (left & kIndexMask)), a.experts - 1);
          const float l_left = logit_of(e_left), b_left = biased ? a.bias[e_left] : 0.f;
#pragma unroll
          for (int j = 0; j < VPL; ++j) {
            const int e = l8 * VPL + j;
            if (key[j] < left && float(left_value - (key[j] >> kIndexBits)) <= margin && e < a.experts) {
              const float l = logit_of(e);
              other |= l > -INFINITY && !(l == l_left && (!biased || a.bias[e] == b_left));
            }
          }
        }
        const unsigned others = __ballot_sync(kAll, other);
        unsure |= deep && (((close_lanes | others) >> (lane & 24)) & 255u) != 0;
      }
    }
    const unsigned unsure_lanes = __ballot_sync(kAll, unsure);
    const bool done = (((unsure_lanes | close_lanes) >> (lane & 24)) & 255u) == 0;

    // weights, as in write_weights
    float w = 0.f;
    if (a.renormalize) {
      const float most = eight_max_nan(logit);
      if (!sigmoid) {
        w = has_pick ? expf(logit - most) : 0.f;
      } else {
        const float t = expf(-fabsf(logit));
        float numerator = logit < 0.f ? t : 1.f;
        if (most < 0.f) numerator = expf(logit - most);
        w = has_pick ? __fdividef(numerator, 1.f + t) : 0.f;
      }
      w = __fdividef(w, eight_sum(w));
    } else {
      w = sigmoid ? sigmoid_of(logit) : __fdividef(expf(logit - top), total);
    }
    if (has_pick && done && token < a.tokens) {
      a.weights[token * a.top_k + l8] = w * a.scale;
      a.chosen[token * a.top_k + l8] = expert;
    }
    __syncwarp();
    if ((unsure_lanes | close_lanes) != 0) {
      for (int t = 0; t < 4; ++t) {
        const unsigned close_t = (close_lanes >> (8 * t)) & 255u;
        if (first + t >= a.tokens) break;
        if (((unsure_lanes >> (8 * t)) & 255u) != 0) {
          route_token_apart<T, GROUPED ? kAnyGroups : kNoGroups>(a, first + t, scratch[GROUPED ? warp : 0]);
        } else if (close_t != 0) {
          const int source = 8 * t + (lane & 7);
          Picks p{__shfl_sync(kAll, expert, source), __shfl_sync(kAll, logit, source)};
          const uint32_t left_t = __shfl_sync(kAll, left, 8 * t);
          const bool joins = ((edge_lanes >> (8 * t)) & 255u) != 0;  // the one left behind takes part
          if (joins && lane == a.top_k) {
            p.expert = int(kIndexMask - (left_t & kIndexMask));
            p.logit = float(*reinterpret_cast<const T*>(staged[warp][buf] + t * kRowBytes + p.expert / VPL * kLaneBytes +
                                                        p.expert % VPL * int(sizeof(T))));
          }
          refine_apart<T>(a, first + t, __shfl_sync(kAll, top, 8 * t), __shfl_sync(kAll, total, 8 * t), p,
                          a.top_k + (joins ? 1 : 0));
        }
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Returns false for what the kernel does not take.
template <typename T, int VPL>
bool launch_many_vpl(Args a, cudaStream_t s) {
  const int lanes = a.group_size / VPL;
  const bool grouped = a.num_groups > 1;
  if (grouped && (a.group_size % VPL != 0 || (lanes & (lanes - 1)) != 0)) return false;
  a.many_lanes_log = 0;
  while (grouped && (1 << a.many_lanes_log) < lanes) ++a.many_lanes_log;
  const int64_t blocks = (a.tokens + 4 * kManyWarps - 1) / (4 * kManyWarps), places = (VPL <= 16 ? 6 : 4) * 148;
  const int grid = int(blocks < places ? blocks : places);
  if (grouped) route_many_kernel<T, VPL, true><<<grid, kManyWarps * 32, 0, s>>>(a);
  else route_many_kernel<T, VPL, false><<<grid, kManyWarps * 32, 0, s>>>(a);
  return true;
}

template <typename T>
bool launch_many(const Args& a, cudaStream_t s) {
  constexpr int kSize = int(sizeof(T));
  if (a.tokens < (a.num_groups > 1 ? 16384 : 8192) || a.top_k > kManyMaxPicks || a.experts < 32 || a.experts > 256 ||
      (a.experts * kSize) % 16 != 0 || (a.ld * kSize) % 16 != 0 || reinterpret_cast<uintptr_t>(a.logits) % 16 != 0)
    return false;
  if (a.experts <= 64) return launch_many_vpl<T, 8>(a, s);
  if (a.experts <= 128) return launch_many_vpl<T, 16>(a, s);
  if (a.experts <= 192) return launch_many_vpl<T, 24>(a, s);
  return launch_many_vpl<T, 32>(a, s);
}

template <typename T, int VPL>
int launch_vpl(Args& a, cudaStream_t s) {
  constexpr int kBytes = VPL * int(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
  a.vec = a.experts % VPL == 0 && reinterpret_cast<uintptr_t>(a.logits) % kWord == 0 && (a.ld * int64_t(sizeof(T))) % kWord == 0;
  const int64_t blocks = (a.tokens + kWarps - 1) / kWarps;
  const int64_t places = int64_t(kResident<VPL>) * 148;
  const int grid = int(blocks < places ? blocks : places);
  const int lanes = a.group_size / VPL;
  if (a.num_groups == 1) {
    route_experts_kernel<T, VPL, kNoGroups><<<grid, kWarps * 32, 0, s>>>(a);
  } else if (a.group_size % VPL == 0 && (lanes & (lanes - 1)) == 0) {
    a.lanes_log = 0;
    while ((1 << a.lanes_log) < lanes) ++a.lanes_log;
    route_experts_kernel<T, VPL, kLaneGroups><<<grid, kWarps * 32, 0, s>>>(a);
  } else {
    route_experts_kernel<T, VPL, kAnyGroups><<<grid, kWarps * 32, 0, s>>>(a);
  }
  return launch_status();
}

template <typename T>
int launch(Args& a, cudaStream_t s) {
  if (launch_many<T>(a, s)) return launch_status();
  if (a.experts <= 32) return launch_vpl<T, 1>(a, s);
  if (a.experts <= 64) return launch_vpl<T, 2>(a, s);
  if (a.experts <= 128) return launch_vpl<T, 4>(a, s);
  if (a.experts <= 256) return launch_vpl<T, 8>(a, s);
  if (a.experts <= 512) return launch_vpl<T, 16>(a, s);
  return launch_vpl<T, 32>(a, s);
}

}  // namespace route
}  // namespace hb200

extern "C" int hb200_moe_route_experts(const hb200_route_args* args, void* stream) {
  using namespace hb200;
  if (!args) return HB200_ERR_INVALID_ARGUMENT;
  const auto [logits, bias, weights, chosen, tokens, experts, ld, top_k, num_groups, top_groups, group_top, logits_dtype, scoring,
              renormalize, scale] = *args;
  if (!logits || !weights || !chosen || tokens < 0 || experts < 1 || experts > 1024 || ld < 0) return HB200_ERR_INVALID_ARGUMENT;
  if (top_k < 1 || top_k > 32 || num_groups < 1 || num_groups > 32 || experts % num_groups != 0 || top_groups < 1 ||
      top_groups > num_groups || top_k > top_groups * (experts / num_groups))
    return HB200_ERR_INVALID_ARGUMENT;
  if (group_top < 1 || group_top > 2 || (group_top > 1 && experts / num_groups < 2)) return HB200_ERR_INVALID_ARGUMENT;
  if (logits_dtype < 0 || logits_dtype > 2 || scoring < 0 || scoring > 1) return HB200_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return HB200_OK;
  route::Args a{};
  a.logits = logits;
  a.ld = ld;
  a.tokens = tokens;
  a.bias = bias;
  a.weights = weights;
  a.chosen = chosen;
  a.experts = int(experts);
  a.top_k = int(top_k);
  a.sigmoid = scoring == 1;
  a.num_groups = int(num_groups);
  a.top_groups = int(top_groups);
  a.group_top = int(group_top);
  a.group_size = int(experts / num_groups);
  a.renormalize = renormalize != 0;
  a.scale = scale;
  a.lanes_log = 0;
  while ((num_groups << (a.lanes_log + 1)) <= 32) ++a.lanes_log;
  while (int(a.group_low) < a.num_groups - 1) a.group_low = 2 * a.group_low + 1;
  a.group_inv = uint32_t(((1 << 20) + a.group_size - 1) / a.group_size);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_dtype == 0) return route::launch<__nv_bfloat16>(a, s);
  if (logits_dtype == 1) return route::launch<__half>(a, s);
  return route::launch<float>(a, s);
}

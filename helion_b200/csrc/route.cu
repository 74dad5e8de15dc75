// Routing of tokens to experts: scores, a balance bias, expert groups, top-k and the weights, one warp per token.
//
//   score_e  = softmax(logits)_e or sigmoid(logit_e)                         (0 for a masked expert, logit -inf)
//   choice_e = score_e + bias_e, or the logit itself without a bias          (same order as the score, and exact)
//   groups: a group's score is the sum of its best group_top live choices (with group_top = 2 and no bias: of its
//           best scores); the best top_groups groups stay
//   picks:  the top_k best choices of the experts that stay, equal choices by ascending index, masked experts last
//   weights: the picks' scores (without the bias), divided by their sum if asked for, times scale
//
// Which experts come out is decided as in exact arithmetic: choices computed in fp32 are off by less than `margin`
// (below), and a row in which two neighbouring picks, or the last group that stays and the first that goes, are
// closer than that is decided again in 64 bits.  Bound by issue and latency, not by bytes.
#include "common.cuh"

namespace hb200 {
namespace route {

constexpr int kWarps = 8;

struct Args {
  const void* logits;
  int64_t ld, tokens;
  const float* bias;  // [experts] or nullptr
  float* weights;
  int64_t* chosen;
  int experts, top_k, sigmoid, num_groups, top_groups, group_top, group_size, renormalize;
  float scale;
};

// Order-preserving keys: larger value, larger key; 0 = not to be picked (any more), 1 = masked.  -0 counts as +0.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long long key_of(double v) {
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return u ^ (static_cast<unsigned long long>(static_cast<long long>(u) >> 63) | (1ull << 63));
}
__device__ __forceinline__ double value_of(unsigned long long k) {
  return __longlong_as_double(static_cast<long long>((k >> 63) ? k ^ (1ull << 63) : ~k));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

template <typename R> struct KeyOf;
template <> struct KeyOf<float> { using type = uint32_t; };
template <> struct KeyOf<double> { using type = unsigned long long; };

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <typename R>
__device__ __forceinline__ R sigmoid_of(R v) {
  const R e = exp_of(v < R(0) ? v : -v);
  return (v < R(0) ? e : R(1)) / (R(1) + e);
}

template <typename R>
__device__ __forceinline__ R warp_total(R v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Picks {
  int expert;   // lane r holds pick r
  float logit;
  bool unsure;  // two values that decide the result are closer than the arithmetic can tell
};

template <typename T, int VPL>
__device__ __forceinline__ void load_row(const Args& a, int64_t token, int lane, float (&l)[VPL], float (&b)[VPL]) {
  const T* row = static_cast<const T*>(a.logits) + token * a.ld;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = lane * VPL + j;
    l[j] = e < a.experts ? float(row[e]) : -INFINITY;
    b[j] = (a.bias != nullptr && e < a.experts) ? a.bias[e] : 0.f;
  }
}

// top, total: the row's largest logit and sum of exp(logit - top) (softmax only)
template <typename R, int VPL>
__device__ __forceinline__ Picks choose(const Args& a, int lane, const float (&l)[VPL], const float (&b)[VPL], float top, R total) {
  using Key = typename KeyOf<R>::type;
  constexpr bool kExact = sizeof(R) == 8;
  constexpr unsigned kAll = 0xffffffffu;
  const bool biased = a.bias != nullptr;
  // fp32 scores are off by at most 5 units of 2^-24 (sigmoid: one exponential, one addition, one division of values
  // up to 1) or 17 (softmax: rounding of logit - top scaled by score, the sum's own error); the sum with the bias
  // adds half a unit in the last place of the choice.  Twice that separates two choices, rounded up.
  const R base = a.sigmoid ? R(1.0 / (1 << 20)) : R(1.0 / (1 << 18));
  auto margin = [&](R v) { return base + (v < R(0) ? -v : v) * R(1.0 / (1 << 22)); };
  auto score = [&](float logit) -> R {
    return a.sigmoid ? sigmoid_of(R(logit)) : exp_of(R(logit) - R(top)) / total;
  };

  Key key[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = lane * VPL + j;
    const bool live = l[j] > -INFINITY;
    R choice = R(l[j]);
    if (biased) choice = (live ? score(l[j]) : R(0)) + R(b[j]);
    key[j] = e >= a.experts ? Key(0) : (live && choice > R(-INFINITY)) ? key_of(choice) : Key(1);
  }
  bool unsure = false;

  if (a.num_groups > 1) {
    R mine = R(-INFINITY);
    for (int g = 0; g < a.num_groups; ++g) {
      const int lo = g * a.group_size, hi = lo + a.group_size;
      Key m1 = 0, m2 = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int e = lane * VPL + j;
        if (e >= lo && e < hi) {
          if (key[j] > m1) { m2 = m1; m1 = key[j]; } else if (key[j] > m2) { m2 = key[j]; }
        }
      }
      const Key best = warp_max(m1);
      R s = R(-INFINITY);
      if (best > Key(1)) {
        const bool of_scores = a.group_top > 1 && !biased;
        s = of_scores ? score(float(value_of(best))) : R(value_of(best));
        if (a.group_top > 1) {
          const int at = __ffs(__ballot_sync(kAll, m1 == best)) - 1;
          const Key next = warp_max(lane == at ? m2 : m1);
          if (next > Key(1)) s += of_scores ? score(float(value_of(next))) : R(value_of(next));
        }
      }
      if (lane == g) mine = s;
    }
    int before = 0;
    for (int g = 0; g < a.num_groups; ++g) {
      const R other = __shfl_sync(kAll, mine, g);
      before += other > mine || (other == mine && g < lane);
    }
    const bool stays = lane < a.num_groups && before < a.top_groups;
    const unsigned kept = __ballot_sync(kAll, stays);
    if (!kExact && (biased || a.group_top > 1) && a.top_groups < a.num_groups) {
      const Key last = ~warp_max(stays ? Key(~key_of(mine)) : Key(0));
      const Key first = warp_max(lane < a.num_groups && !stays ? key_of(mine) : Key(0));
      const R lv = R(value_of(last)), fv = R(value_of(first));
      if (fv > R(-INFINITY) && lv - fv <= R(2) * margin(lv)) unsure = true;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = lane * VPL + j;
      if (e < a.experts && !((kept >> (e / a.group_size)) & 1u)) key[j] = 0;
    }
  }

  Picks p{0, -INFINITY, false};
  Key prev = 0;
  float prev_l = 0.f, prev_b = 0.f;
  const int rounds = a.top_k + (!kExact && biased ? 1 : 0);  // one more to compare the last pick with what it left behind
  for (int r = 0; r < rounds; ++r) {
    Key m = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) m = key[j] > m ? key[j] : m;
    const Key best = warp_max(m);
    const int at = __ffs(__ballot_sync(kAll, m == best)) - 1;
    int e = 0;
    float pl = 0.f, pb = 0.f;
    if (lane == at) {
      bool found = false;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        if (!found && key[j] == best) {
          found = true;
          key[j] = 0;
          e = lane * VPL + j;
          pl = l[j];
          pb = b[j];
        }
      }
    }
    e = __shfl_sync(kAll, e, at);
    pl = __shfl_sync(kAll, pl, at);
    if (!kExact && biased) {
      pb = __shfl_sync(kAll, pb, at);
      if (r > 0 && best > Key(1)) {
        const R hi = R(value_of(prev)), lo = R(value_of(best));
        if (hi - lo <= margin(hi) && !(pl == prev_l && pb == prev_b)) unsure = true;
      }
      prev = best;
      prev_l = pl;
      prev_b = pb;
    }
    if (lane == r && r < a.top_k) {
      p.expert = e;
      p.logit = pl;
    }
  }
  p.unsure = unsure;
  return p;
}

template <typename T, int VPL>
__device__ __noinline__ Picks choose_exactly(const Args& a, int64_t token, int lane) {
  float l[VPL], b[VPL];
  load_row<T, VPL>(a, token, lane, l, b);
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < VPL; ++j) top = fmaxf(top, l[j]);
  top = hb200::warp_max(top);
  double total = 0.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (l[j] > -INFINITY) total += exp(double(l[j]) - double(top));
    total = warp_total(total);
  }
  return choose<double, VPL>(a, lane, l, b, top, total);
}

template <typename T, int VPL>
__global__ void __launch_bounds__(kWarps * 32)
route_experts_kernel(const __grid_constant__ Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t step = int64_t(gridDim.x) * kWarps;
  for (int64_t token = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); token < a.tokens; token += step) {
    float l[VPL], b[VPL];
    load_row<T, VPL>(a, token, lane, l, b);
    // A NaN (or, under softmax, an infinite logit) spoils the row's scores: its weights come out as NaN.
    bool spoilt = false;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      spoilt |= l[j] != l[j] || b[j] != b[j] || (!a.sigmoid && l[j] == INFINITY);
      top = fmaxf(top, l[j]);
    }
    spoilt = __any_sync(0xffffffffu, spoilt);
    top = hb200::warp_max(top);
    float total = 0.f;
    if (!a.sigmoid) {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (l[j] > -INFINITY) total += expf(l[j] - top);
      total = warp_total(total);
    }
    Picks p = choose<float, VPL>(a, lane, l, b, top, total);
    if (p.unsure && !spoilt) p = choose_exactly<T, VPL>(a, token, lane);

    // Weights.  Renormalised ones are ratios of scores: they are formed relative to the largest pick, so that picks
    // far below the row's largest logit (a bias or a group can choose them) keep their ratios.
    const bool live = lane < a.top_k && p.logit > -INFINITY;
    float w = 0.f;
    if (a.renormalize) {
      const float best = hb200::warp_max(live ? p.logit : -INFINITY);
      if (live) {
        if (!a.sigmoid) w = expf(p.logit - best);
        else if (p.logit >= 0.f) w = 1.f / (1.f + expf(-p.logit));
        else w = expf(p.logit - fminf(best, 0.f)) / (1.f + expf(p.logit));
      }
      const float sum = warp_total(w);
      if (live) w = w / sum;
    } else if (live) {
      w = a.sigmoid ? sigmoid_of(p.logit) : expf(p.logit - top) / total;
    }
    w = spoilt ? NAN : w * a.scale;
    if (lane < a.top_k) {
      a.weights[token * a.top_k + lane] = w;
      a.chosen[token * a.top_k + lane] = p.expert;
    }
  }
}

template <typename T>
int launch(const Args& a, cudaStream_t s) {
  const int64_t blocks = (a.tokens + kWarps - 1) / kWarps;
  const int grid = int(blocks < 148 * 8 ? blocks : 148 * 8);
#define HB200_ROUTE(V) route_experts_kernel<T, V><<<grid, kWarps * 32, 0, s>>>(a)
  if (a.experts <= 32) HB200_ROUTE(1);
  else if (a.experts <= 64) HB200_ROUTE(2);
  else if (a.experts <= 128) HB200_ROUTE(4);
  else if (a.experts <= 256) HB200_ROUTE(8);
  else if (a.experts <= 512) HB200_ROUTE(16);
  else HB200_ROUTE(32);
#undef HB200_ROUTE
  return launch_status();
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_dtype == 0) return route::launch<__nv_bfloat16>(a, s);
  if (logits_dtype == 1) return route::launch<__half>(a, s);
  return route::launch<float>(a, s);
}

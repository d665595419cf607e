// A router's choice with the experts in groups: logits [rows, experts] to every row's `top` experts and their weights.
//
//   score   softmax over all experts or the sigmoid of each logit
//   pick    score + bias (the bias counts for the choice alone); a pick that is not a number counts as minus infinity
//   groups  `groups` runs of experts of equal length; a group's score is the sum of its `group_best` (1 or 2) largest picks; the
//           `top_groups` groups with the largest scores are open
//   choice  the `top` largest picks of open groups, largest first; ties go to the lower index, of groups and of experts
//   weight  the chosen scores, divided by (their sum + norm_eps) if `renormalize`, times `scale`
//
// Which of two picks is larger may hang on their last bits, and a choice is whole numbers: it is that of 64-bit scores.  Where nothing is added to
// the scores, their order is the logits' own and those are compared.  Otherwise the row is chosen by 32-bit scores.  Where two neighbours in that order
// are nearer than the scores' error, the chosen experts and those behind them as near are put in the order of their 64-bit scores; a softmax, and a
// row where the last open group and the first closed one are as near, is chosen once more by 64-bit scores of all experts.
//
// A warp per row, expert lane + 32 j the lane's j-th.  Picks lie in registers as unsigned numbers of the same order, so that a largest one of the
// warp is one instruction (redux.sync; two for 64 bits) and its lowest index another.  Bound by a row's chain of instructions, some 1,600 for 256
// experts in 8 groups: 64 rows 6.4 us, 8,192 rows 18.4 to 22 (their bytes take 1.4); a row that is chosen once more takes 8 to 11 more by itself.
#include "common.cuh"
#include <math.h>

SRB_DEFINE_LAST_ERROR()
SRB_DEFINE_PDL_SWITCH()

#define ROUTE_MAX_EXPERTS 1024
#define ROUTE_MAX_TOP 32
#define ROUTE_MAX_GROUPS 32
#define ROUTE_WARPS 4
#define ROUTE_SOFTMAX 0
#define ROUTE_SIGMOID 1
#define ALL 0xffffffffu

struct GroupRule {
  int experts, top, groups, top_groups, group_best, scoring, renormalize;
  float scale, norm_eps;
  int per_group;
  unsigned group_factor;         // e * group_factor >> 20 is e / per_group, for e < 1024
};

// Numbers in the order of the reals that they stand for; 0 is below all of them.
__device__ __forceinline__ unsigned route_key(float v) {
  const unsigned u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float route_value(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long route_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double route_value(unsigned long long key) {
  return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}
__device__ __forceinline__ unsigned route_most(unsigned key) { return __reduce_max_sync(ALL, key); }
__device__ __forceinline__ unsigned long long route_most(unsigned long long key) {
  const unsigned high = __reduce_max_sync(ALL, (unsigned)(key >> 32));
  const unsigned low = __reduce_max_sync(ALL, (unsigned)(key >> 32) == high ? (unsigned)key : 0u);
  return (unsigned long long)high << 32 | low;
}

// Whether 32-bit numbers do not tell which of two picks (or sums of two) is larger, `above` being the larger one of them.  `by_logit`: they are the logits
// themselves, whose order is that of the scores but where 64-bit scores are alike: both 0; sigmoids near 1 (2^-53 apart is e^-36, and logits
// below 36 that are 1 apart differ by more); logits so near 0 that the exponential does not see them apart (below 1e-5 two may be nearer
// than 9e-13, and an argument of up to 700 is good to 2e-13).  Otherwise they are off by at most 1.75 2^-22 of the scores that went in (the
// exponential by 1.5 2^-23 of itself, over all floats 1.28 2^-23 at most; the sum under the division, the division, the sum with the bias and that of two
// picks by 2^-24 each), or, in a softmax, 2^-16: its exponential's argument is off by 2^-24 of its size, which is below 104 where anything is left of
// the score (6.2e-6 of it), the sum by 2^-24 for each of up to 37 additions (2.2e-6) and as much as its terms (the largest ones have small
// arguments: 1e-6), the quick division by 2^-22.  Beside that by 2^-126, where 32 bits end.
__device__ __forceinline__ bool route_near(float above, float below, float bias_most, float most, bool by_logit, int scoring) {
  if (by_logit)
    return !(below - (scoring == ROUTE_SOFTMAX ? most : 0.f) > -700.f) || (fabsf(above) < 1e-5f && above - below < 9e-13f) ||
           (scoring == ROUTE_SIGMOID && above > 16.f && !(above - below >= 1.f && below <= 36.f));
  const float room = fmaf(fabsf(above) + fabsf(below) + 2.f * bias_most, scoring == ROUTE_SOFTMAX ? 1.5258789e-5f : 4.3e-7f, 2.3509887e-38f);
  return !(above - below > room);
}

// The score of a group whose largest two picks each lane has among its own.
template <typename Key>
__device__ __forceinline__ Key route_group_score(Key first, Key second, int group_best, int lane) {
  const Key best = route_most(first);
  auto sum = route_value(best);
  if (group_best == 2) {
    const int owner = __ffs(__ballot_sync(ALL, first == best)) - 1;
    sum += route_value(route_most(lane == owner ? second : first));
  }
  return route_key(sum == sum ? sum : (decltype(sum))-INFINITY);
}

// The lane k < top gets the k-th choice by 32-bit scores; it holds unless `near_groups` or `near`: then the groups are in doubt, or the order of the
// `count` experts that the lanes k < count hold, which go on behind the top ones as long as neighbours are near (32 of them: there may be
// more).  `most` and `sum`: of a softmax.  `picks`: room for a key of every expert.
template <int PER>
__device__ __forceinline__ int route_choose(const float (&z)[PER], const float* __restrict__ bias, const GroupRule& rule, float most, float sum,
                                            unsigned* picks, int lane, bool& near_groups, bool& near, int& count) {
  const bool by_logit = !bias && (rule.group_best == 1 || rule.groups == rule.top_groups);
  unsigned key[PER];
  float bias_most = 0.f;
  const float over_sum = __fdividef(1.0f, sum);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    float pick = z[j] + 0.f;                                 // -0 lies where 0 does
    if (!by_logit) pick = rule.scoring == ROUTE_SOFTMAX ? expf(pick - most) * over_sum : 1.0f / (1.0f + expf(-pick));
    if (bias && e < rule.experts) {
      const float b = __ldg(bias + e);
      bias_most = fmaxf(bias_most, fabsf(b));
      pick += b;
    }
    key[j] = e < rule.experts ? route_key(pick == pick ? pick : -INFINITY) : 0u;
  }
  if (bias) bias_most = __uint_as_float(__reduce_max_sync(ALL, __float_as_uint(bias_most)));
  near_groups = near = false;
  if (rule.groups > rule.top_groups) {
    const int per_group = rule.per_group;
    unsigned mine = 0u;                                      // the score of group `lane`
    if (per_group % 32 == 0) {
      // a group is some of the registers, of all lanes
      int g = 0, end = per_group;
      unsigned first = 0u, second = 0u;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        second = max(second, min(first, key[j]));
        first = max(first, key[j]);
        if (32 * (j + 1) == end) {
          const unsigned score = route_group_score(first, second, rule.group_best, lane);
          if (lane == g) mine = score;
          first = second = 0u;
          end = ++g < rule.groups ? end + per_group : 0;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (lane + 32 * j < rule.experts) picks[lane + 32 * j] = key[j];
      __syncwarp();
      for (int g = 0; g < rule.groups; ++g) {
        unsigned first = 0u, second = 0u;
        for (int i = lane; i < per_group; i += 32) {
          const unsigned v = picks[g * per_group + i];
          second = max(second, min(first, v));
          first = max(first, v);
        }
        const unsigned score = route_group_score(first, second, rule.group_best, lane);
        if (lane == g) mine = score;
      }
      __syncwarp();
    }
    unsigned open = 0u;
    float first = 0.f, last = 0.f;
    for (int k = 0; k < rule.top_groups; ++k) {
      const unsigned best = route_most(mine);
      if (k == 0) first = route_value(best);
      const int g = __ffs(__ballot_sync(ALL, mine == best)) - 1;
      open |= 1u << g;
      if (lane == g) mine = 0u;
      last = route_value(best);
    }
    near_groups = route_near(last, route_value(route_most(mine)), 2.f * bias_most, most, by_logit, rule.scoring);
    // logits that are all alike are in their order
    if (near_groups && by_logit) {
      const float lowest = route_value(__reduce_min_sync(ALL, mine ? mine : ALL));
      near_groups = !(first == lowest && lowest > -INFINITY);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j < rule.experts && !((open >> ((unsigned)(lane + 32 * j) * rule.group_factor >> 20)) & 1u)) key[j] = 0u;
  }
  int choice = 0;
  float last = 0.f;
  for (count = 0;; ++count) {
    unsigned mine = 0u;
#pragma unroll
    for (int j = 0; j < PER; ++j) mine = max(mine, key[j]);
    const unsigned best = route_most(mine);
    if (best == 0u) break;                                   // all are taken
    const float value = route_value(best);
    const bool close = count > 0 && route_near(last, value, bias_most, most, by_logit, rule.scoring);
    if (count >= rule.top && !close) break;
    near |= close && !(by_logit && last == value && value > -INFINITY);      // equal logits are in their order, a NaN is not at minus infinity's
    if (count == 32) {                                       // no lane is left: the run goes on as it is, or is in doubt
      unsigned lowest = ALL;
#pragma unroll
      for (int j = 0; j < PER; ++j) lowest = min(lowest, key[j] ? key[j] : ALL);
      near |= close && __reduce_min_sync(ALL, lowest) != best;
      break;
    }
    last = value;
    unsigned index = 0x7fffffffu;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if (key[j] == best) index = (unsigned)(lane + 32 * j);
    index = __reduce_min_sync(ALL, index);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (index == (unsigned)(lane + 32 * j)) key[j] = 0u;
    if (lane == count) choice = (int)index;
  }
  return choice;
}

// The same by 64-bit scores, for the few rows that need it: loops over the keys in shared memory, with little code laid out flat, since a warp that comes
// here waits for the instructions to be fetched.
__device__ __noinline__ int route_choose_exactly(const float* __restrict__ z, const float* __restrict__ bias, const GroupRule& rule, unsigned long long* keys,
                                                 int lane) {
  double most = -INFINITY, sum = 0.0;
  if (rule.scoring == ROUTE_SOFTMAX) {
#pragma unroll 1
    for (int e = lane; e < rule.experts; e += 32) most = fmax(most, (double)z[e]);
    most = route_value(route_most(route_key(most)));
#pragma unroll 1
    for (int e = lane; e < rule.experts; e += 32) sum += exp((double)z[e] - most);
#pragma unroll 1
    for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(ALL, sum, offset);
  }
#pragma unroll 4
  for (int e = lane; e < rule.experts; e += 32) {
    const bool softmax = rule.scoring == ROUTE_SOFTMAX;
    const double power = exp(softmax ? (double)z[e] - most : -(double)z[e]);
    double pick = (softmax ? power : 1.0) / (softmax ? sum : 1.0 + power);
    if (bias) pick += (double)bias[e];
    keys[e] = route_key(pick == pick ? pick : (double)-INFINITY);
  }
  __syncwarp();
  if (rule.groups > rule.top_groups) {
    unsigned long long mine = 0;
#pragma unroll 1
    for (int g = 0; g < rule.groups; ++g) {
      unsigned long long first = 0, second = 0;
#pragma unroll 1
      for (int i = lane; i < rule.per_group; i += 32) {
        const unsigned long long v = keys[g * rule.per_group + i];
        second = max(second, min(first, v));
        first = max(first, v);
      }
      const unsigned long long score = route_group_score(first, second, rule.group_best, lane);
      if (lane == g) mine = score;
    }
    unsigned open = 0u;
#pragma unroll 1
    for (int k = 0; k < rule.top_groups; ++k) {
      const int g = __ffs(__ballot_sync(ALL, mine == route_most(mine))) - 1;
      open |= 1u << g;
      if (lane == g) mine = 0;
    }
    __syncwarp();
#pragma unroll 1
    for (int e = lane; e < rule.experts; e += 32)
      if (!((open >> ((unsigned)e * rule.group_factor >> 20)) & 1u)) keys[e] = 0;
  }
  int choice = 0;
#pragma unroll 1
  for (int k = 0; k < rule.top; ++k) {
    unsigned long long best = 0;
    unsigned index = 0x7fffffffu;
#pragma unroll 4
    for (int e = lane; e < rule.experts; e += 32)
      if (keys[e] > best) { best = keys[e]; index = (unsigned)e; }
    index = __reduce_min_sync(ALL, best == route_most(best) ? index : 0x7fffffffu);
    if (lane == (int)(index & 31u)) keys[index] = 0;         // the lane that reads it
    if (lane == k) choice = (int)index;
  }
  return choice;
}

// The lanes k < count hold experts whose sigmoids go into the order of their 64-bit picks.
__device__ __noinline__ int route_reorder(const float* __restrict__ z, const float* __restrict__ bias, int choice, int count, int lane) {
  unsigned long long key = 0;
  if (lane < count) {
    double pick = 1.0 / (1.0 + exp(-(double)z[choice]));
    if (bias) pick += (double)bias[choice];
    key = route_key(pick == pick ? pick : (double)-INFINITY);
  }
  int rank = 0, ordered = choice;
  for (int i = 0; i < count; ++i) {
    const unsigned long long other = __shfl_sync(ALL, key, i);
    const int expert = __shfl_sync(ALL, choice, i);          // by all lanes, before anything depends on the lane
    rank += other > key || (other == key && expert < choice) ? 1 : 0;
  }
  for (int i = 0; i < count; ++i) {
    const int at = __shfl_sync(ALL, rank, i), expert = __shfl_sync(ALL, choice, i);
    if (lane == at) ordered = expert;
  }
  return ordered;
}

// The weight of the lane's choice in 64 bits, `argument` being that of the exponential.
__device__ __noinline__ float route_far_weight(double argument, float sum, const GroupRule& rule, int lane) {
  double weight = 0.0;
  if (lane < rule.top) weight = rule.scoring == ROUTE_SOFTMAX ? exp(argument) / (double)sum : 1.0 / (1.0 + exp(-argument));
  if (rule.renormalize) {
    double all = weight;
#pragma unroll 1
    for (int offset = 16; offset > 0; offset >>= 1) all += __shfl_xor_sync(ALL, all, offset);
    weight /= all + (double)rule.norm_eps;
  }
  return (float)(weight * (double)rule.scale);
}

template <int PER>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, PER <= 8 ? 10 : 1)
route_groups_kernel(const float* __restrict__ logits, size_t pitch, int rows, const float* __restrict__ bias, GroupRule rule,
                    int* __restrict__ chosen, float* __restrict__ weights) {
  extern __shared__ unsigned long long route_shared[];       // [warps][experts]
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * ROUTE_WARPS + warp;
  if (row >= rows) return;
  unsigned long long* shared = route_shared + (size_t)warp * rule.experts;
  const float* from = logits + (size_t)row * pitch;
  float z[PER];
  float most = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    z[j] = lane + 32 * j < rule.experts ? from[lane + 32 * j] : -INFINITY;
    most = fmaxf(most, z[j]);
  }
  if (rule.scoring == ROUTE_SOFTMAX) {
    most = route_value(route_most(route_key(most)));
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j < rule.experts) sum += expf(z[j] - most);
    sum = srb_warp_sum(sum);
  }
  bool near_groups, near;
  int count;
  int choice = route_choose<PER>(z, bias, rule, most, sum, reinterpret_cast<unsigned*>(shared), lane, near_groups, near, count);
  // a few neighbours in doubt are put in order among themselves; groups, more of them, and a softmax, whose sum has all experts in it (and no scores
  // where something is not finite), take the whole row
  if (near_groups || (near && (count == 32 || rule.scoring == ROUTE_SOFTMAX)) || (rule.scoring == ROUTE_SOFTMAX && !(sum < INFINITY)))
    choice = route_choose_exactly(from, bias, rule, shared, lane);
  else if (near)
    choice = route_reorder(from, bias, choice, count, lane);
  // the chosen scores, a lane each; where 32 bits do not hold one (below e^-87), in 64: divided by their sum they may be anything
  const float logit = lane < rule.top ? from[choice] : 0.f;
  float weight = 0.f;
  if (lane < rule.top) weight = rule.scoring == ROUTE_SOFTMAX ? expf(logit - most) / sum : 1.0f / (1.0f + expf(-logit));
  if (__any_sync(ALL, lane < rule.top && weight < 1e-37f)) {
    weight = route_far_weight(rule.scoring == ROUTE_SOFTMAX ? (double)logit - (double)most : (double)logit, sum, rule, lane);
  } else {
    if (rule.renormalize) weight /= srb_warp_sum(weight) + rule.norm_eps;
    weight *= rule.scale;
  }
  if (lane < rule.top) {
    chosen[(size_t)row * rule.top + lane] = choice;
    weights[(size_t)row * rule.top + lane] = weight;
  }
}

extern "C" int srb_route_groups(const float* logits, long long pitch, int rows, int experts, const float* bias, int top, int groups,
                                int top_groups, int group_best, int scoring, int renormalize, float scale, float norm_eps, int* chosen,
                                float* weights, void* stream) {
  if (experts <= 0 || experts > ROUTE_MAX_EXPERTS) SRB_FAIL("route_groups: %d experts are outside 1 .. %d", experts, ROUTE_MAX_EXPERTS);
  if (groups <= 0 || groups > ROUTE_MAX_GROUPS || experts % groups) SRB_FAIL("route_groups: %d experts in %d groups", experts, groups);
  if (top_groups <= 0 || top_groups > groups) SRB_FAIL("route_groups: %d open groups of %d", top_groups, groups);
  if (group_best < 1 || group_best > 2 || group_best > experts / groups)
    SRB_FAIL("route_groups: a group's score by its %d best of %d", group_best, experts / groups);
  if (top <= 0 || top > ROUTE_MAX_TOP || top > experts / groups * top_groups)
    SRB_FAIL("route_groups: %d chosen experts are outside 1 .. min(%d, %d)", top, experts / groups * top_groups, ROUTE_MAX_TOP);
  if (scoring != ROUTE_SOFTMAX && scoring != ROUTE_SIGMOID) SRB_FAIL("route_groups: unknown scoring %d", scoring);
  if (pitch < experts) SRB_FAIL("route_groups: rows of the logits overlap");
  if (rows <= 0) return SRB_OK;
  const int per_group = experts / groups;
  const GroupRule rule{experts, top, groups, top_groups, group_best, scoring, renormalize, scale, norm_eps, per_group, (1u << 20) / per_group + 1u};
  auto kernel = experts <= 64 ? route_groups_kernel<2> : experts <= 256 ? route_groups_kernel<8> : route_groups_kernel<32>;
  SRB_CUDA_CALL(srb_launch(kernel, dim3((rows + ROUTE_WARPS - 1) / ROUTE_WARPS), dim3(32 * ROUTE_WARPS), (size_t)ROUTE_WARPS * experts * 8,
                           (cudaStream_t)stream, logits, (size_t)pitch, rows, bias, rule, chosen, weights));
  return SRB_OK;
}

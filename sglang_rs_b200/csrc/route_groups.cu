// A router's choice with the experts in groups: logits [rows, experts] to every row's `top` experts and their weights.
//
//   score   softmax over all experts or the sigmoid of each logit
//   pick    score + bias (the bias counts for the choice alone); a pick that is not a number counts as minus infinity
//   groups  `groups` runs of experts of equal length; a group's score is the sum of its `group_best` (1 or 2) largest picks; the
//           `top_groups` groups with the largest scores are open
//   choice  the `top` largest picks of open groups, largest first; ties go to the lower index, of groups and of experts
//   weight  the chosen scores, divided by (their sum + norm_eps) if `renormalize`, times `scale`
//
// Which of two picks is larger may hang on their last bits, and a choice is whole numbers: the row is chosen in 32 bits, and once more in 64
// where two neighbours in that order, or the last open group and the first closed one, are nearer than the 32-bit scores' error.
//
// A warp per row.  Picks lie in registers as unsigned numbers of the same order, so that a largest one of the warp is one instruction
// (redux.sync) and its lowest index another.  Bound by instructions: about 700 a row of 256 experts.
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
};

// numbers in the order of floats; 0 is below every float
__device__ __forceinline__ unsigned route_key(float v) {
  const unsigned u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float route_value(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

__device__ __forceinline__ double route_max(double v) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v = fmax(v, __shfl_xor_sync(ALL, v, offset));
  return v;
}

// The row in 64 bits; `picks` is shared memory for its experts.  The lane k < top returns the k-th choice.
__device__ __noinline__ int route_exactly(const float* z, const float* bias, const GroupRule& rule, double* picks, int lane) {
  double most = -INFINITY, sum = 0.0;
  if (rule.scoring == ROUTE_SOFTMAX) {
    for (int e = lane; e < rule.experts; e += 32) most = fmax(most, (double)z[e]);
    most = route_max(most);
    for (int e = lane; e < rule.experts; e += 32) sum += exp((double)z[e] - most);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) sum += __shfl_xor_sync(ALL, sum, offset);
  }
  for (int e = lane; e < rule.experts; e += 32) {
    const double s = rule.scoring == ROUTE_SOFTMAX ? exp((double)z[e] - most) / sum : 1.0 / (1.0 + exp(-(double)z[e]));
    const double pick = bias ? s + (double)bias[e] : s;
    picks[e] = pick == pick ? pick : -INFINITY;
  }
  __syncwarp();
  const int per_group = rule.experts / rule.groups;
  unsigned open = ALL;
  if (rule.groups > rule.top_groups) {
    double mine = -INFINITY;                                 // the score of group `lane`
    if (lane < rule.groups) {
      double first = -INFINITY, second = -INFINITY;
      for (int i = 0; i < per_group; ++i) {
        const double v = picks[lane * per_group + i];
        if (v > first) { second = first; first = v; }
        else if (v > second) second = v;
      }
      mine = rule.group_best == 2 ? first + second : first;
      if (mine != mine) mine = -INFINITY;
    }
    bool left = lane < rule.groups;
    open = 0;
    for (int k = 0; k < rule.top_groups; ++k) {
      const double best = route_max(left ? mine : -INFINITY);
      const int g = __ffs(__ballot_sync(ALL, left && mine == best)) - 1;
      open |= 1u << g;
      left = left && lane != g;
    }
  }
  int choice = 0;
  for (int k = 0; k < rule.top; ++k) {
    double best = -INFINITY;
    int index = 0x7fffffff;
    for (int e = lane; e < rule.experts; e += 32) {
      const double v = picks[e];
      // a taken one is not a number
      if (v == v && ((open >> (e / per_group)) & 1u) && (v > best || index == 0x7fffffff)) { best = v; index = e; }
    }
    const double most_left = route_max(best);
    const int e = (int)__reduce_min_sync(ALL, best == most_left ? (unsigned)index : 0x7fffffffu);
    if (lane == k) choice = e;
    if (lane == 0) picks[e] = __longlong_as_double(0x7ff8000000000000ll);
    __syncwarp();
  }
  return choice;
}

// The scores' relative error in 32 bits is below 2^-19 (the argument of a softmax's exponential is rounded: 2^-24 times its size, which
// is below 24 where the score is above 2^-34; smaller picks are always looked at in 64 bits).
__device__ __forceinline__ bool route_near(float above, float below, float bias_most) {
  const float room = (fabsf(above) + fabsf(below) + 2.f * bias_most) * 1.9073486e-6f;
  return !(above - below > room) || (bias_most == 0.f && below < 5.8207661e-11f);
}

// PER experts a lane: expert lane + 32 j is the lane's j-th.
template <int PER>
__global__ void __launch_bounds__(32 * ROUTE_WARPS)
route_groups_kernel(const float* __restrict__ logits, size_t pitch, int rows, const float* __restrict__ bias, GroupRule rule,
                    int* __restrict__ chosen, float* __restrict__ weights) {
  extern __shared__ double route_shared[];                   // [warps][experts]
  srb_launch_dependents();
  srb_grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * ROUTE_WARPS + warp;
  if (row >= rows) return;
  double* shared = route_shared + (size_t)warp * rule.experts;
  const float* z = logits + (size_t)row * pitch;
  float score[PER];
  float most = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    score[j] = lane + 32 * j < rule.experts ? z[lane + 32 * j] : -INFINITY;
    most = fmaxf(most, score[j]);
  }
  float sum = 1.f;
  if (rule.scoring == ROUTE_SOFTMAX) {
    most = route_value(__reduce_max_sync(ALL, route_key(most)));
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      score[j] = expf(score[j] - most);
      if (lane + 32 * j < rule.experts) sum += score[j];
    }
    sum = srb_warp_sum(sum);
    const float inverse = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] *= inverse;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) score[j] = 1.0f / (1.0f + expf(-score[j]));
  }
  unsigned key[PER];
  float bias_most = 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 32 * j;
    float pick = score[j];
    if (bias && e < rule.experts) {
      const float b = bias[e];
      bias_most = fmaxf(bias_most, fabsf(b));
      pick += b;
    }
    key[j] = e < rule.experts ? route_key(pick == pick ? pick : -INFINITY) : 0u;
  }
  if (bias) bias_most = __uint_as_float(__reduce_max_sync(ALL, __float_as_uint(bias_most)));
  bool near = false;
  if (rule.groups > rule.top_groups) {
    const int per_group = rule.experts / rule.groups;
    unsigned* picks = reinterpret_cast<unsigned*>(shared);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j < rule.experts) picks[lane + 32 * j] = key[j];
    __syncwarp();
    unsigned mine = 0u;                                      // the score of group `lane`
    for (int g = 0; g < rule.groups; ++g) {
      unsigned first = 0u, second = 0u;
      for (int i = lane; i < per_group; i += 32) {
        const unsigned v = picks[g * per_group + i];
        second = max(second, min(first, v));
        first = max(first, v);
      }
      const unsigned best = __reduce_max_sync(ALL, first);
      float group = route_value(best);
      if (rule.group_best == 2) {
        const int owner = __ffs(__ballot_sync(ALL, first == best)) - 1;
        group += route_value(__reduce_max_sync(ALL, lane == owner ? second : first));
      }
      if (lane == g) mine = route_key(group == group ? group : -INFINITY);
    }
    unsigned open = 0u;
    float last = 0.f;
    for (int k = 0; k <= rule.top_groups; ++k) {
      const unsigned best = __reduce_max_sync(ALL, mine);
      const float value = route_value(best);
      if (k == rule.top_groups) {
        near = route_near(last, value, 2.f * bias_most);
        break;
      }
      const int g = __ffs(__ballot_sync(ALL, mine == best)) - 1;
      open |= 1u << g;
      if (lane == g) mine = 0u;
      last = value;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j < rule.experts && !((open >> ((lane + 32 * j) / per_group)) & 1u)) key[j] = 0u;
    __syncwarp();
  }
  int choice = 0;
  float last = 0.f;
  for (int k = 0; k <= rule.top && !near; ++k) {
    unsigned mine = 0u;
#pragma unroll
    for (int j = 0; j < PER; ++j) mine = max(mine, key[j]);
    const unsigned best = __reduce_max_sync(ALL, mine);
    if (best == 0u) break;                                   // all are taken
    const float value = route_value(best);
    if (k > 0) near = route_near(last, value, bias_most);
    last = value;
    if (k == rule.top) break;
    unsigned index = 0x7fffffffu;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j)
      if (key[j] == best) index = (unsigned)(lane + 32 * j);
    index = __reduce_min_sync(ALL, index);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (index == (unsigned)(lane + 32 * j)) key[j] = 0u;
    if (lane == k) choice = (int)index;
  }
  if (near) choice = route_exactly(z, bias, rule, shared, lane);
  // the chosen scores once more, a lane each
  float weight = 0.f;
  if (lane < rule.top)
    weight = rule.scoring == ROUTE_SOFTMAX ? expf(z[choice] - most) / sum : 1.0f / (1.0f + expf(-z[choice]));
  if (rule.renormalize) weight /= srb_warp_sum(weight) + rule.norm_eps;
  if (lane < rule.top) {
    chosen[(size_t)row * rule.top + lane] = choice;
    weights[(size_t)row * rule.top + lane] = weight * rule.scale;
  }
}

extern "C" int srb_route_groups(const float* logits, long long pitch, int rows, int experts, const float* bias, int top, int groups,
                                int top_groups, int group_best, int scoring, int renormalize, float scale, float norm_eps, int* chosen,
                                float* weights, void* stream) {
  if (rows <= 0) return SRB_OK;
  if (experts <= 0 || experts > ROUTE_MAX_EXPERTS) SRB_FAIL("route_groups: %d experts are outside 1 .. %d", experts, ROUTE_MAX_EXPERTS);
  if (groups <= 0 || groups > ROUTE_MAX_GROUPS || experts % groups) SRB_FAIL("route_groups: %d experts in %d groups", experts, groups);
  if (top_groups <= 0 || top_groups > groups) SRB_FAIL("route_groups: %d open groups of %d", top_groups, groups);
  if (group_best < 1 || group_best > 2 || group_best > experts / groups)
    SRB_FAIL("route_groups: a group's score by its %d best of %d", group_best, experts / groups);
  if (top <= 0 || top > ROUTE_MAX_TOP || top > experts / groups * top_groups)
    SRB_FAIL("route_groups: %d chosen experts are outside 1 .. min(%d, %d)", top, experts / groups * top_groups, ROUTE_MAX_TOP);
  if (scoring != ROUTE_SOFTMAX && scoring != ROUTE_SIGMOID) SRB_FAIL("route_groups: unknown scoring %d", scoring);
  if (pitch < experts) SRB_FAIL("route_groups: rows of the logits overlap");
  const GroupRule rule{experts, top, groups, top_groups, group_best, scoring, renormalize, scale, norm_eps};
  auto kernel = experts <= 64 ? route_groups_kernel<2> : experts <= 256 ? route_groups_kernel<8> : route_groups_kernel<32>;
  SRB_CUDA_CALL(srb_launch(kernel, dim3((rows + ROUTE_WARPS - 1) / ROUTE_WARPS), dim3(32 * ROUTE_WARPS), (size_t)ROUTE_WARPS * experts * 8,
                           (cudaStream_t)stream, logits, (size_t)pitch, rows, bias, rule, chosen, weights));
  SRB_LAUNCH_CHECK("route_groups");
  return SRB_OK;
}

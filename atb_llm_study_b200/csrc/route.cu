// Grouped router selection (the published DeepSeek-V2 / V3 gates): scores of
// the experts from fp32 logits, a balance bias that only the choice sees, the
// best groups of experts, the top-k experts among them and their weights.
//
//   x = logits clamped to the finite range (NaN: the lowest value)
//   s = softmax(x) or sigmoid(x);  c = s + bias;  group score = the sum of a
//   group's 1 or 2 largest c;  experts outside the topk_groups best groups are
//   out;  the top_k largest c (ties, as between groups, to the lower index);
//   weight = s (renormalised over the chosen, 0 where they sum to 0) * scale
//
// The choice is that of the definition in 64 bits: it is made on fp32 scores
// whose error is bounded, and a token with two candidates nearer to one another
// than that bound is chosen again on scores in double.  Without a bias the
// experts are ranked by the logits themselves, which needs no bound.
#include <float.h>
#include <math.h>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 8;
constexpr int kWarps = 4;

struct RouteParams {
  const float* logits;
  int64_t ld;
  const float* bias;
  int64_t T;
  int E, k, sigmoid, G, gs, lpg_shift, keep, best, renorm;
  float scale;
  int32_t* ids;
  float* wts;
};

__device__ __forceinline__ float wmax(float v) { return warp_max(v); }
__device__ __forceinline__ double wmax(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F wsum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// One warp chooses one token's experts with scores of type F.  Lane l of group
// g's 2^lpg_shift lanes holds PER consecutive experts, so lanes, and values
// within a lane, are in expert order.  Returns whether every decision was
// clear of the scores' error (double: always).
template <typename F, int PER>
__device__ __forceinline__ bool choose(const RouteParams& p, int64_t t, int lane) {
  constexpr bool kFloat = sizeof(F) == 4;
  const int lpg = 1 << p.lpg_shift;
  const int g = lane >> p.lpg_shift, l = lane & (lpg - 1);
  const int e0 = g * p.gs + l * PER;
  const int n = g < p.G ? min(max(p.gs - l * PER, 0), PER) : 0;  // experts in this lane
  F s[PER], c[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float x = -FLT_MAX;
    if (i < n) x = fminf(fmaxf(p.logits[t * p.ld + e0 + i], -FLT_MAX), FLT_MAX);  // NaN gives -FLT_MAX
    c[i] = (F)x;
  }
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = i < n ? F(1) / (F(1) + exp_of(-c[i])) : F(0);
  } else {
    F m = F(-FLT_MAX);
#pragma unroll
    for (int i = 0; i < PER; ++i) m = c[i] > m ? c[i] : m;
    m = wmax(m);
    F sum = F(0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = i < n ? exp_of(c[i] - m) : F(0);
      sum += s[i];
    }
    sum = wsum(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = s[i] / sum;
  }
  // Bounds for fp32 scores.  expf is within 2 ulp and its argument within half
  // an ulp of x - max (s |x - max| <= 0.37), the sum of up to 256 terms within
  // 21 roundings (16 in the lane, 5 over the lanes), the division within half
  // an ulp: 1.8e-6 of the largest score covers an error, twice that and the
  // roundings of the biased sums a difference of two.
  F tol = F(0);
  bool clear = true;
  if (kFloat && (p.bias || p.best > 1)) {
    F top = F(0);
#pragma unroll
    for (int i = 0; i < PER; ++i) top = s[i] > top ? s[i] : top;
    tol = F(4e-6) * wmax(top);
  }
  const bool ranked_by_score = p.bias != nullptr;
  if (ranked_by_score) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const F v = i < n ? s[i] + (F)p.bias[e0 + i] : F(0);
      c[i] = v == v ? v : F(-FLT_MAX);
    }
  }
  bool in = n > 0;  // this lane's group is kept
  if (p.keep < p.G) {
    // the group's two largest scores, over its lanes
    const F low = F(-INFINITY);
    F a = low, b = low;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const F v = i < n ? (p.best > 1 && !ranked_by_score ? s[i] : c[i]) : low;
      const F lo = a < v ? a : v;
      a = a < v ? v : a;
      b = b < lo ? lo : b;
    }
    for (int o = 1; o < lpg; o <<= 1) {
      const F oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      const F lo = a < oa ? a : oa, hb = b < ob ? ob : b;
      a = a < oa ? oa : a;
      b = lo < hb ? hb : lo;
    }
    const F score = p.best > 1 ? a + b : a;
    const F size = (a < 0 ? -a : a) + (p.best > 1 ? (b < 0 ? -b : b) : F(0));
    const F near = (p.best > 1 ? 2 * tol : tol) + F(3.6e-7) * size;
    int rank = 0;
    bool doubt = false;
    for (int h = 0; h < p.G; ++h) {
      const F other = __shfl_sync(0xffffffffu, score, h << p.lpg_shift);
      rank += other > score || (other == score && h < g);
      const F d = other > score ? other - score : score - other;
      doubt |= h != g && d <= near;
    }
    in = in && rank < p.keep;
    if (kFloat && tol > F(0)) clear = !__any_sync(0xffffffffu, doubt && g < p.G);
  }
  int mine = 0x7fffffff;  // lane j < k: the j-th choice
  F mine_s = F(0), sum = F(0), before = F(0);
  unsigned taken = 0;
  // one round more than k, when it exists: the best that was not chosen
#pragma unroll 1
  for (int j = 0; j <= p.k; ++j) {
    F bv = F(0), bs = F(0);
    int bi = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (in && i < n && !(taken >> i & 1u) && (bi < 0 || c[i] > bv)) {
        bv = c[i];
        bs = s[i];
        bi = i;
      }
    }
    const unsigned have = __ballot_sync(0xffffffffu, bi >= 0);
    if (!have) break;
    const F top = wmax(bi >= 0 ? bv : F(-INFINITY));
    const int from = __ffs(__ballot_sync(0xffffffffu, bi >= 0 && bv == top)) - 1;
    if (kFloat && ranked_by_score && j > 0 && before - top <= tol + F(1.2e-7) * (top < 0 ? -top : top)) clear = false;
    before = top;
    if (j == p.k) break;
    const int e = __shfl_sync(0xffffffffu, e0 + bi, from);
    const F w = __shfl_sync(0xffffffffu, bs, from);
    if (lane == from) taken |= 1u << bi;
    if (lane == j) {
      mine = e;
      mine_s = w;
    }
    sum += w;
  }
  if (kFloat && p.renorm && sum < F(1e-30)) clear = false;  // weights below fp32's range
  if (kFloat && !clear) return false;
  if (lane < p.k) {
    p.ids[t * p.k + lane] = mine;
    const F w = p.renorm ? (sum > F(0) ? mine_s / sum : F(0)) : mine_s;
    p.wts[t * p.k + lane] = (float)(w * (F)p.scale);
  }
  return true;
}

template <int PER>
__device__ __noinline__ void choose_in_double(const RouteParams& p, int64_t t, int lane) {
  choose<double, PER>(p, t, lane);
}

template <int PER>
__global__ void __launch_bounds__(kWarps * 32) topk_grouped_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  if (!choose<float, PER>(p, t, lane)) choose_in_double<PER>(p, t, lane);
}

}  // namespace

extern "C" int b200_moe_topk_grouped(const float* logits, int64_t ld, const float* bias, int64_t T, int num_experts,
                                     int top_k, int scoring, int num_groups, int topk_groups, int group_top,
                                     int renormalize, float scale, int32_t* topk_ids, float* topk_weights,
                                     b200_stream_t stream) {
  if (!logits || !topk_ids || !topk_weights || T < 0 || num_experts <= 0 || ld < num_experts ||
      (scoring != B200_SCORE_SOFTMAX && scoring != B200_SCORE_SIGMOID))
    return B200_ERROR_INVALID_PARAM;
  if (num_groups <= 0 || num_experts % num_groups || topk_groups <= 0 || topk_groups > num_groups ||
      (group_top != 1 && group_top != 2) || group_top > num_experts / num_groups)
    return B200_ERROR_INVALID_PARAM;
  if (top_k <= 0 || top_k > kMaxTopK || top_k > topk_groups * (num_experts / num_groups))
    return B200_ERROR_INVALID_PARAM;
  for (const void* q : {(const void*)logits, (const void*)bias, (const void*)topk_ids, (const void*)topk_weights})
    if ((uintptr_t)q & 3u) return B200_ERROR_INVALID_PARAM;
  if (num_experts > kMaxExperts || num_groups > 32) return B200_ERROR_UNSUPPORTED;
  if (T > (int64_t)INT32_MAX) return B200_ERROR_UNSUPPORTED;
  if (T == 0) return B200_OK;
  RouteParams p{};
  p.logits = logits;
  p.ld = ld;
  p.bias = bias;
  p.T = T;
  p.E = num_experts;
  p.k = top_k;
  p.sigmoid = scoring == B200_SCORE_SIGMOID;
  // without a limit on the groups they do not matter: all experts are one group
  p.G = topk_groups < num_groups ? num_groups : 1;
  p.keep = topk_groups < num_groups ? topk_groups : 1;
  p.gs = num_experts / p.G;
  p.best = p.G > 1 ? group_top : 1;
  p.renorm = renormalize != 0;
  p.scale = scale;
  p.ids = topk_ids;
  p.wts = topk_weights;
  while ((p.G << (p.lpg_shift + 1)) <= 32) ++p.lpg_shift;
  const int per = (p.gs + (1 << p.lpg_shift) - 1) >> p.lpg_shift;
  const dim3 grid((unsigned)((T + kWarps - 1) / kWarps));
  if (per <= 1) launch_kernel(topk_grouped_kernel<1>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 2) launch_kernel(topk_grouped_kernel<2>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 4) launch_kernel(topk_grouped_kernel<4>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 8) launch_kernel(topk_grouped_kernel<8>, grid, kWarps * 32, 0, stream, p);
  else launch_kernel(topk_grouped_kernel<16>, grid, kWarps * 32, 0, stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

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
// than that bound is chosen again on scores in double.
//
// One warp a token, four a CTA.  The bytes (4 E T read) are not what bounds it
// but the comparisons' half-rate integer pipe, and the choice in double beside
// them: 16384 x 256, 4 of 8 groups, top-8 with a bias 21.2 us (17.8 MB, 2.7 us at
// the copy rate), 15.1 in a build that has no choice in double (32 registers
// instead of 80), for the 0.12 % of tokens that take it; 16384 x 64 ungrouped 10.5
// us (7.9 without), 4099 x 160 7.0 us, 64 x 64 2.1 us.  All tokens in double take
// 46 us for the first, as a batch of nothing but ties does.
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
  int vec;  // the lanes' runs of logits (and biases) are whole, aligned float4s
  int32_t* ids;
  float* wts;
};

// ---------------------------------------------------------------------------
// One warp per token.  Lane l of group g's 2^lpg_shift lanes holds PER
// consecutive experts, so lanes, and values within a lane, are in expert order.
// ---------------------------------------------------------------------------
struct Slot {
  int g, e0, n;  // group, first expert and number of experts of this lane
};

template <int PER>
__device__ __forceinline__ Slot slot_of(const RouteParams& p, int lane) {
  const int l = lane & ((1 << p.lpg_shift) - 1);
  Slot s;
  s.g = lane >> p.lpg_shift;
  s.e0 = s.g * p.gs + l * PER;
  s.n = s.g < p.G ? min(max(p.gs - l * PER, 0), PER) : 0;
  return s;
}

// To the finite range (NaN: the lowest value), -0 to 0.
__device__ __forceinline__ float clamp_logit(float x) { return fminf(fmaxf(x, -FLT_MAX), FLT_MAX) + 0.f; }

template <int PER>
__device__ __forceinline__ void load_run(float v[PER], const float* src, const Slot& s, int vec, float fill) {
  if (PER % 4 == 0 && vec) {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i)
      if (s.n > 0) {
        const float4 f = *reinterpret_cast<const float4*>(src + s.e0 + 4 * i);
        v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
      } else {
        v[4 * i] = v[4 * i + 1] = v[4 * i + 2] = v[4 * i + 3] = fill;
      }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = i < s.n ? src[s.e0 + i] : fill;
  }
}

// fp32 values as unsigned integers of the same order (0: below every value),
// the lowest bits replaced by a tag.
__device__ __forceinline__ uint32_t to_key(float v, uint32_t tag_bits, uint32_t tag) {
  const uint32_t b = __float_as_uint(v);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (o & ~tag_bits) | tag;
}
__device__ __forceinline__ float from_key(uint32_t k, uint32_t tag_bits) {
  k &= ~tag_bits;
  return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// Descending (Batcher's odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_desc(uint32_t k[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j <= N - 1 - q; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = k[i + j], y = k[i + j + q];
            k[i + j] = max(x, y);
            k[i + j + q] = min(x, y);
          }
}

// Without the scaling that keeps subnormal arguments and results (they are far
// below the bounds here).
__device__ __forceinline__ float exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The choice on fp32 scores; false (nothing written) when two candidates of a
// decision are nearer than the scores' error.
//
// What is compared carries a tag in its low bits, so one 32-bit maximum over
// the warp gives value and place: log2(PER) bits among experts (the place in
// the lane), 5 among groups (whose choice is then checked on the whole values).
// Cutting b bits moves a value by less than 2^(b-23) of itself.  Two equal values
// are always in doubt, so ties are settled in double, by index.
//
// Error of a score (exp_fast: 2 + 1.2 |x| ulp of e^x).  Sigmoid: the quotient's
// ulp, half an ulp of the sum 1 + e^-x, and the exponential's error times
// s (1 - s), at most 0.6 ulp: 2.4e-7, a difference of two 5e-7.  Softmax, in
// units of the largest score: the term's own 2 ulp of 1, the sum's 21 roundings
// and its terms' errors (1.6e-6 where every term counts), the product: 2.5e-6, a
// difference of two 5e-6.
template <int PER>
__device__ __forceinline__ bool choose_fast(const RouteParams& p, int64_t t, int lane) {
  constexpr int kTagBits = PER <= 1 ? 0 : PER <= 2 ? 1 : PER <= 4 ? 2 : PER <= 8 ? 3 : 4;
  constexpr uint32_t kTag = (1u << kTagBits) - 1u, kGroupTag = 31u;
  // 2^(bits - 23), and the half ulps of the two values compared
  constexpr float kCut = (float)(1 << kTagBits) * 0x1p-23f + 1.2e-7f;
  const Slot sl = slot_of<PER>(p, lane);
  const float* lg = p.logits + t * p.ld;
  float c[PER];
  load_run<PER>(c, lg, sl, p.vec, -FLT_MAX);
#pragma unroll
  for (int i = 0; i < PER; ++i) c[i] = clamp_logit(c[i]);
  const bool pair_groups = p.keep < p.G && p.best > 1;
  const bool by_score = p.bias != nullptr;  // without a bias experts are ranked by their logits
  float m = 0.f, inv = 1.f, top = 1.f;      // softmax: the largest logit, 1 / sum, the largest score
  if (!p.sigmoid) {
    m = c[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) m = fmaxf(m, c[i]);
    m = from_key(__reduce_max_sync(0xffffffffu, to_key(m, 0u, 0u)), 0u);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += i < sl.n ? exp_fast(c[i] - m) : 0.f;
    inv = rcp_fast(warp_sum(sum));
    top = inv;
  }
  float s[PER];  // scores, where anything is ranked by them
  if (by_score || pair_groups) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = p.sigmoid ? rcp_fast(1.f + exp_fast(-c[i])) : exp_fast(c[i] - m) * inv;
  }
  if (by_score) {
    float b[PER];
    load_run<PER>(b, p.bias, sl, p.vec, 0.f);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = fmaxf(s[i] + b[i], -FLT_MAX);
    }
  }
  const float tol = by_score || pair_groups ? (p.sigmoid ? 5e-7f : 5e-6f * top) : 0.f;
  bool in = true, clear = true;
  if (p.keep < p.G) {
    // the group's one or two largest, over its lanes
    float a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float v = i < sl.n ? (p.best > 1 && !by_score ? s[i] : c[i]) : -INFINITY;
      b = fmaxf(b, fminf(a, v));
      a = fmaxf(a, v);
    }
    for (int o = 1; o < (1 << p.lpg_shift); o <<= 1) {
      const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      b = fmaxf(fminf(a, oa), fmaxf(b, ob));
      a = fmaxf(a, oa);
    }
    const float score = p.best > 1 ? a + b : a;
    // score -+ err holds the group's score in 64 bits: the errors of its one or
    // two scores, and where anything but logits is compared the roundings of the
    // biased scores, of their sum and of score -+ err (half an ulp each).  Those
    // are relative to the terms, which can cancel, so every group has a bound of
    // its own, whatever its rank.
    const float err = (p.best > 1 ? tol : 0.5f * tol) +
                      (tol > 0.f ? 2.4e-7f * (p.best > 1 ? fabsf(a) + fabsf(b) : fabsf(a)) : 0.f);
    uint32_t key = sl.g < p.G ? to_key(score, kGroupTag, 31u - sl.g) : 0u;
    in = false;
    for (int j = 0; j < p.keep; ++j) {
      const uint32_t best = __reduce_max_sync(0xffffffffu, key);
      if (key == best) {
        in = true;
        key = 0u;
      }
    }
    // every group that is kept against the best that another may be (a sum below
    // fp32's range is below -3e38, too)
    const float most = in || sl.g >= p.G ? -INFINITY : score == -INFINITY ? -3e38f : score + err;
    const float other = from_key(__reduce_max_sync(0xffffffffu, to_key(most, 0u, 0u)), 0u);
    clear = __all_sync(0xffffffffu, !in || score - err > other);
  }
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = in && i < sl.n ? to_key(c[i], kTag, kTag - i) : 0u;
  sort_desc<PER>(key);
  uint32_t mine = 0;  // lane j: the j-th choice's key, and the lane that holds it
  int from_lane = 0;
  for (int j = 0; j <= p.k; ++j) {  // one more than is chosen: the best that is not
    const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
    const int from = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
    if (lane == j) {
      mine = best;
      from_lane = from;
    }
    if (lane == from) {
#pragma unroll
      for (int i = 0; i + 1 < PER; ++i) key[i] = key[i + 1];
      key[PER - 1] = 0u;
    }
  }
  {
    // every choice against the next; a next that does not exist has key 0
    const uint32_t next = __shfl_down_sync(0xffffffffu, mine, 1);
    const float x = from_key(mine, kTag), y = from_key(next, kTag);
    const bool apart = lane >= p.k || next == 0u || x - y > (by_score ? tol + kCut * fabsf(x) : 0.f);
    clear = clear && __all_sync(0xffffffffu, apart);
  }
  if (!clear) return false;
  // lane j < k: the j-th choice and its weight, from its logit
  int e = 0;
  float w = 0.f;
  if (lane < p.k) {
    const Slot from = slot_of<PER>(p, from_lane);
    e = from.e0 + (int)(kTag - (mine & kTag));
    const float x = clamp_logit(lg[e]);
    w = p.sigmoid ? 1.f / (1.f + expf(-x)) : expf(x - m) * inv;
  }
  if (p.renorm) {
    float sum = w;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (__shfl_sync(0xffffffffu, sum, 0) < 1e-30f) return false;  // scores below fp32's range
    w = w / sum;
  }
  if (lane < p.k) {
    p.ids[t * p.k + lane] = e;
    p.wts[t * p.k + lane] = w * p.scale;
  }
  return true;
}

// Doubles as unsigned integers of the same order (-0 as 0).
__device__ __forceinline__ uint64_t to_key64(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ uint64_t warp_max64(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}

// The choice on scores in double (experts without a bias by their logits).
template <int PER>
__device__ __noinline__ void choose_exact(const RouteParams& p, int64_t t, int lane) {
  const Slot sl = slot_of<PER>(p, lane);
  const double low = -INFINITY;
  double s[PER], c[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) c[i] = i < sl.n ? clamp_logit(p.logits[t * p.ld + sl.e0 + i]) : low;
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = 1.0 / (1.0 + exp(-c[i]));
  } else {
    float mf = -FLT_MAX;  // (logits are fp32 values)
#pragma unroll
    for (int i = 0; i < PER; ++i) mf = fmaxf(mf, (float)c[i]);
    const double m = warp_max(mf);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = exp(c[i] - m);
      sum += s[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum = 1.0 / sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] *= sum;
  }
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i < sl.n) c[i] = s[i] + (double)p.bias[sl.e0 + i];
      if (!(c[i] >= -DBL_MAX)) c[i] = i < sl.n ? -DBL_MAX : low;
    }
  }
  bool in = sl.n > 0;
  if (p.keep < p.G) {
    double a = low, b = low;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double v = i < sl.n ? (p.best > 1 && !p.bias ? s[i] : c[i]) : low;
      b = fmax(b, fmin(a, v));
      a = fmax(a, v);
    }
    for (int o = 1; o < (1 << p.lpg_shift); o <<= 1) {
      const double oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      b = fmax(fmin(a, oa), fmax(b, ob));
      a = fmax(a, oa);
    }
    uint64_t key = sl.g < p.G ? to_key64(p.best > 1 ? a + b : a) : 0u;
    in = false;
    for (int j = 0; j < p.keep; ++j) {
      const uint64_t top = warp_max64(key);
      const int from = __ffs(__ballot_sync(0xffffffffu, key == top)) - 1;  // of equals the lowest group
      if (sl.g == from >> p.lpg_shift) {
        in = sl.n > 0;
        key = 0u;
      }
    }
  }
  uint64_t key[PER];  // 0: not to be chosen (no value's key)
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = in && i < sl.n ? to_key64(c[i]) : 0u;
  int mine = 0;  // lane j < k: the j-th choice
  double mine_s = 0.0, sum = 0.0;
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    uint64_t bk = key[0];
    double bs = s[0];
    int bi = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i) {
      if (key[i] > bk) {  // the first of equals
        bk = key[i];
        bs = s[i];
        bi = i;
      }
    }
    const uint64_t top = warp_max64(bk);
    const int from = __ffs(__ballot_sync(0xffffffffu, bk == top)) - 1;
    const int e = __shfl_sync(0xffffffffu, sl.e0 + bi, from);
    const double w = __shfl_sync(0xffffffffu, bs, from);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane == from && i == bi) key[i] = 0u;
    if (lane == j) {
      mine = e;
      mine_s = w;
    }
    sum += w;
  }
  if (lane < p.k) {
    p.ids[t * p.k + lane] = mine;
    if (p.renorm) mine_s = sum > 0.0 ? mine_s / sum : 0.0;
    p.wts[t * p.k + lane] = (float)(mine_s * (double)p.scale);
  }
}

template <int PER>
__global__ void __launch_bounds__(kWarps * 32) topk_grouped_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  if (!choose_fast<PER>(p, t, lane)) choose_exact<PER>(p, t, lane);
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
  const int held = per <= 4 ? 4 : 8;
  p.vec = p.gs == held << p.lpg_shift && ld % 4 == 0 && ((uintptr_t)logits & 15u) == 0 && ((uintptr_t)bias & 15u) == 0;
  const dim3 grid((unsigned)((T + kWarps - 1) / kWarps));
  if (per <= 1) launch_kernel(topk_grouped_kernel<1>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 2) launch_kernel(topk_grouped_kernel<2>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 4) launch_kernel(topk_grouped_kernel<4>, grid, kWarps * 32, 0, stream, p);
  else if (per <= 8) launch_kernel(topk_grouped_kernel<8>, grid, kWarps * 32, 0, stream, p);
  else launch_kernel(topk_grouped_kernel<16>, grid, kWarps * 32, 0, stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

// Logits of a decode step made ready for the choice of a token: penalties for
// repeated tokens, biases, a grammar's mask, and the greedy token.
//
// Per row, with said(v) the times token v occurs behind the prompt:
//   x = logit(v); if v occurs at all: x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * said(v); if said(v): x -= presence
//   x += the biases listed for v; -inf where the mask has no bit for v.
//
// A row's logits are read and written once (4 bytes a token, 600 KB at 151936),
// so memory bounds a batch; one row is bound by latency.  What makes the pass
// more than a copy is knowing which tokens occur: the vocabulary is split over
// the CTAs of a cluster, and each keeps a word for every token of its part in
// shared memory: the count, and a bit for the prompt.  Each CTA walks the whole
// history (16 KB for 4000 tokens, from L2) and counts what falls into its part
// with integer atomics in shared memory, whose result has no order.  A table in
// global memory instead would cost 4 bytes a token to clear, and to read once.
// Tokens that occur nowhere, by far the most, are copied; the few others are
// computed in double (operation by operation, nothing contracted), so that the
// greedy token is that of the definition and not of 32-bit roundings.
#include <math.h>

#include <algorithm>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int kThreads = 512;
constexpr uint32_t kTopBit = 1u << 31;  // of a history word: in the prompt; of a bias word: listed more than once
constexpr int kMaxSmem = 224 * 1024;

struct LogitsParams {
  const __nv_bfloat16* logits;
  int64_t ld;
  int64_t vocab;
  int chunk;  // tokens a CTA, a multiple of 32
  const int32_t* history;
  int64_t history_ld;
  const int32_t* prompt_lens;
  const int32_t* lens;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int32_t* bias_offsets;
  const int32_t* bias_ids;
  const float* bias_values;
  const uint32_t* mask;
  int64_t mask_ld;
  int64_t num_masks;
  const int32_t* mask_rows;
  __nv_bfloat16* out;
  int64_t ldo;
  int64_t* next;
  int vec;  // 16-byte accesses: rows and pointers are aligned
  unsigned* err;
};

// The better of two candidates: the larger value, the lower token on ties.  Token INT64_MAX: none.
struct Best {
  double v;
  int64_t i;
};
B200_DEV Best better(const Best& a, const Best& b) { return b.v > a.v || (b.v == a.v && b.i < a.i) ? b : a; }

B200_DEV uint64_t cluster_load8(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// HIST / BIAS: the call has a history / a bias list, and shared memory holds the words for it.
template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t words[];
  __shared__ Best warp_best[kThreads / 32];
  __shared__ Best cta_best;
  uint32_t* seen = words;                           // [chunk] times behind the prompt | kTopBit
  uint32_t* lead = words + (HIST ? p.chunk : 0);    // [chunk] entries from its first to the list's end | kTopBit
  pdl_trigger();
  const int ctas = (int)cluster_size();
  const int64_t row = blockIdx.x / ctas;
  const int64_t lo = (int64_t)cluster_rank() * p.chunk;
  const int n = (int)max((int64_t)0, min((int64_t)p.chunk, p.vocab - lo));
  const int tid = threadIdx.x;
  const int kinds = (HIST ? 1 : 0) + (BIAS ? 1 : 0);
  for (int i = tid; i < kinds * p.chunk / 4; i += kThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  pdl_wait();

  if (HIST) {
    int len = p.lens[row], prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
    if (len < 0 || len > p.history_ld || prompt < 0 || prompt > len) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
      len = (int)min((int64_t)max(len, 0), p.history_ld);
      prompt = min(max(prompt, 0), len);
    }
    const int32_t* h = p.history + row * p.history_ld;
#pragma unroll 4
    for (int i = tid; i < len; i += kThreads) {
      const int64_t at = (int64_t)h[i] - lo;
      if (at >= 0 && at < n) {
        if (i < prompt) atomicOr(&seen[at], kTopBit);
        else atomicAdd(&seen[at], 1u);
      } else if (h[i] < 0 || h[i] >= p.vocab) {
        raise_error(p.err, DEV_ERR_BAD_INDEX);
      }
    }
  }
  int b0 = 0, nb = 0;
  if (BIAS) {
    b0 = p.bias_offsets[row];
    nb = p.bias_offsets[row + 1] - b0;
    if (b0 < 0 || nb < 0) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
      b0 = nb = 0;
    }
    // a token's first entry leads: it is worth the most counted from the end
    for (int i = tid; i < nb; i += kThreads) {
      const int64_t id = p.bias_ids[b0 + i], at = id - lo;
      if (at >= 0 && at < n) atomicMax(&lead[at], (uint32_t)(nb - i));
      else if (id < 0 || id >= p.vocab) raise_error(p.err, DEV_ERR_BAD_INDEX);
    }
    __syncthreads();
    for (int i = tid; i < nb; i += kThreads) {
      const int64_t at = (int64_t)p.bias_ids[b0 + i] - lo;
      if (at >= 0 && at < n && (lead[at] & ~kTopBit) != (uint32_t)(nb - i)) atomicOr(&lead[at], kTopBit);
    }
  }
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int64_t m = p.mask_rows ? p.mask_rows[row] : row;
    if (m >= p.num_masks || m < -1) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
    } else if (m >= 0) {
      mask = p.mask + m * p.mask_ld;
    }
  }
  const bool rep = HIST && p.repetition, frq = HIST && p.frequency, prs = HIST && p.presence;
  const double repetition = rep ? (double)p.repetition[row] : 1.0;
  const double frequency = frq ? (double)p.frequency[row] : 0.0;
  const double presence = prs ? (double)p.presence[row] : 0.0;
  __syncthreads();

  const __nv_bfloat16* in = p.logits + row * p.ld + lo;
  __nv_bfloat16* out = p.out ? p.out + row * p.ldo + lo : nullptr;
  float plain_v = -INFINITY;  // untouched tokens are bf16 values: compared as they are
  int64_t plain_i = INT64_MAX;
  Best best{-INFINITY, INT64_MAX};

  // token `at` of this CTA's part with logit x, words w and l: its value; a touched token's goes into `best`
  auto process = [&](int at, float x, uint32_t w, uint32_t l) -> __nv_bfloat16 {
    double v = (double)x;
    if (HIST && w) {
      if (rep) v = v > 0 ? __ddiv_rn(v, repetition) : __dmul_rn(v, repetition);
      const uint32_t said = w & ~kTopBit;
      if (frq) v = __dsub_rn(v, __dmul_rn(frequency, (double)said));
      if (prs && said) v = __dsub_rn(v, presence);
    }
    if (BIAS && l) {
      const int first = nb - (int)(l & ~kTopBit);
      double sum = (double)p.bias_values[b0 + first];
      for (int i = l & kTopBit ? first + 1 : nb; i < nb; ++i)  // a token listed twice: in the order of the list
        if (p.bias_ids[b0 + i] == p.bias_ids[b0 + first]) sum = __dadd_rn(sum, (double)p.bias_values[b0 + i]);
      v = __dadd_rn(v, sum);
    }
    if (v > best.v) best = {v, lo + at};
    return __double2bfloat16(v);
  };

  if (p.vec) {
    for (int c = tid; c < n / 8; c += kThreads) {
      const uint4 raw = reinterpret_cast<const uint4*>(in)[c];
      uint32_t w[8], l[8], touched = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = l[i] = 0;
      if (HIST) {
        *reinterpret_cast<uint4*>(w) = reinterpret_cast<const uint4*>(seen)[2 * c];
        *reinterpret_cast<uint4*>(w + 4) = reinterpret_cast<const uint4*>(seen)[2 * c + 1];
      }
      if (BIAS) {
        *reinterpret_cast<uint4*>(l) = reinterpret_cast<const uint4*>(lead)[2 * c];
        *reinterpret_cast<uint4*>(l + 4) = reinterpret_cast<const uint4*>(lead)[2 * c + 1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) touched |= (w[i] | l[i]) ? 1u << i : 0u;
      const uint32_t allowed = mask ? (mask[(lo >> 5) + (c >> 2)] >> ((c & 3) * 8)) & 0xffu : 0xffu;
      float f[8];
      unpack8(raw, f);
      uint4 res = raw;
      if (touched == 0 && allowed == 0xffu) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (f[i] > plain_v) {
            plain_v = f[i];
            plain_i = lo + c * 8 + i;
          }
      } else {
        __nv_bfloat16* r = reinterpret_cast<__nv_bfloat16*>(&res);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!((allowed >> i) & 1u)) {
            r[i] = __float2bfloat16_rn(-INFINITY);
          } else if ((touched >> i) & 1u) {
            r[i] = process(c * 8 + i, f[i], w[i], l[i]);
          } else if (f[i] > plain_v) {
            plain_v = f[i];
            plain_i = lo + c * 8 + i;
          }
        }
      }
      if (out) reinterpret_cast<uint4*>(out)[c] = res;
    }
  }
  // rows that 16-byte accesses do not fit, and the last few tokens of those that they do
  for (int at = (p.vec ? n & ~7 : 0) + tid; at < n; at += kThreads) {
    __nv_bfloat16 r = in[at];
    const float x = bf2f(r);
    const uint32_t w = HIST ? seen[at] : 0, l = BIAS ? lead[at] : 0;
    if (mask && !((mask[(lo + at) >> 5] >> (at & 31)) & 1u)) {
      r = __float2bfloat16_rn(-INFINITY);
    } else if (w | l) {
      r = process(at, x, w, l);
    } else if (x > plain_v) {
      plain_v = x;
      plain_i = lo + at;
    }
    if (out) out[at] = r;
  }
  if (!p.next) return;

  best = better(best, Best{(double)plain_v, plain_i});
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
  if ((tid & 31) == 0) warp_best[tid >> 5] = best;
  __syncthreads();
  if (tid < 32) {
    best = tid < kThreads / 32 ? warp_best[tid] : Best{-INFINITY, INT64_MAX};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)});
    if (tid == 0) cta_best = best;
  }
  cluster_sync();
  if (cluster_rank() == 0 && tid == 0) {
    for (int r = 1; r < ctas; ++r) {
      const uint32_t at = cluster_map(smem_u32(&cta_best), r);
      best = better(best, Best{__longlong_as_double((long long)cluster_load8(at)), (int64_t)cluster_load8(at + 8)});
    }
    p.next[row] = best.i == INT64_MAX ? -1 : best.i;
  }
  cluster_sync();  // the parts stay until they are read
}

template <bool HIST, bool BIAS>
int launch(const LogitsParams& p, int64_t rows, unsigned ctas, cudaStream_t stream) {
  auto k = logits_kernel<HIST, BIAS>;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERROR_UNSUPPORTED;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess ||
        cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    done[dev] = true;
  }
  const size_t smem = (size_t)p.chunk * 4 * ((HIST ? 1 : 0) + (BIAS ? 1 : 0));
  launch_clusters(k, ctas, dim3((unsigned)(rows * ctas)), kThreads, smem, stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

}  // namespace

extern "C" int b200_logits_process(const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                                   const int32_t* history, int64_t history_ld, const int32_t* prompt_lens,
                                   const int32_t* lens, const float* repetition, const float* frequency,
                                   const float* presence, const int32_t* bias_offsets, const int32_t* bias_ids,
                                   const float* bias_values, const uint32_t* mask, int64_t mask_ld, int64_t num_masks,
                                   const int32_t* mask_rows, void* out, int64_t ldo, int64_t* next,
                                   b200_stream_t stream) {
  if (!logits || (!out && !next) || rows < 0 || vocab <= 0 || ld < vocab || (out && ldo < vocab))
    return B200_ERROR_INVALID_PARAM;
  if (out == logits && ldo != ld) return B200_ERROR_INVALID_PARAM;
  const bool hist = history != nullptr, bias = bias_offsets != nullptr;
  if (hist ? (!lens || history_ld <= 0) : (prompt_lens || lens || repetition || frequency || presence))
    return B200_ERROR_INVALID_PARAM;
  if (bias ? (!bias_ids || !bias_values) : (bias_ids || bias_values)) return B200_ERROR_INVALID_PARAM;
  if (mask ? (mask_ld < (vocab + 31) / 32 || num_masks <= 0 || (!mask_rows && num_masks < rows)) : mask_rows != nullptr)
    return B200_ERROR_INVALID_PARAM;
  for (const void* q : {(const void*)history, (const void*)prompt_lens, (const void*)lens, (const void*)repetition,
                        (const void*)frequency, (const void*)presence, (const void*)bias_offsets,
                        (const void*)bias_ids, (const void*)bias_values, (const void*)mask, (const void*)mask_rows})
    if (reinterpret_cast<uintptr_t>(q) & 3u) return B200_ERROR_INVALID_PARAM;
  const uintptr_t pl = reinterpret_cast<uintptr_t>(logits), po = reinterpret_cast<uintptr_t>(out);
  if ((pl & 1u) || (po & 1u) || (reinterpret_cast<uintptr_t>(next) & 7u)) return B200_ERROR_INVALID_PARAM;
  if (rows > INT32_MAX / 16 || vocab > INT32_MAX || history_ld > (int64_t)(kTopBit - 1)) return B200_ERROR_UNSUPPORTED;
  if (rows == 0) return B200_OK;

  // CTAs of a row: 16, or so many that each has 1024 tokens.  (A word or two a
  // token must fit shared memory: 16 CTAs of 224 KB.)
  unsigned ctas = 1;
  while (ctas < 16 && (int64_t)ctas * 1024 < vocab) ctas *= 2;
  const int64_t chunk = ((vocab + ctas - 1) / ctas + 31) / 32 * 32;
  if (chunk * 4 * ((hist ? 1 : 0) + (bias ? 1 : 0)) > kMaxSmem) return B200_ERROR_UNSUPPORTED;
  int dev = 0;
  cudaGetDevice(&dev);
  const int vec = (pl & 15u) == 0 && ld % 8 == 0 && (!out || ((po & 15u) == 0 && ldo % 8 == 0));
  const LogitsParams p{static_cast<const __nv_bfloat16*>(logits), ld, vocab, (int)chunk, history, history_ld,
                       prompt_lens, lens, repetition, frequency, presence, bias_offsets, bias_ids, bias_values, mask,
                       mask_ld, num_masks, mask_rows, static_cast<__nv_bfloat16*>(out), ldo, next, vec,
                       b200::error_word(dev)};
  if (hist) return bias ? launch<true, true>(p, rows, ctas, stream) : launch<true, false>(p, rows, ctas, stream);
  return bias ? launch<false, true>(p, rows, ctas, stream) : launch<false, false>(p, rows, ctas, stream);
}

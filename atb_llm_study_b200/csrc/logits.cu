// Logits of a decode step made ready for the choice of a token: penalties for
// repeated tokens, biases, a grammar's mask, and the greedy token.
//
// Per row, with said(v) the times token v occurs behind the prompt:
//   x = logit(v); if v occurs at all: x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * said(v); if said(v): x -= presence
//   x += the biases listed for v; -inf where the mask has no bit for v.
//
// A row's logits are read and written once (4 bytes a token, 600 KB at 151936),
// so memory bounds a batch in principle, and the few dependent steps between
// lists and logits do in practice.  A row's vocabulary is split over the CTAs of
// a cluster in stripes of 1024 tokens, in turn (vocabularies are sorted by how
// often their tokens occur, so a run of them would have most of the work).  Each marks the tokens of its part that occur in the history or
// among the biases in a bitmap in shared memory (one bit a token), whose prefix
// counts number the marked tokens; per marked token it keeps how often it was
// said, whether the prompt has it and where its biases begin.  All of this is
// whole-number arithmetic, so the order of the atomics does not show.  The sweep
// then copies 16 bytes a thread and masks, leaving marked tokens to a thread
// each: they are computed in double, operation by operation, so that the greedy
// token is that of the definition and not of 32-bit roundings.
//
// Measured at 64 rows of 151936 with up to 4000 tokens of history, 300 biases and
// a mask on every other row, in a replayed graph with L2 flushed: 26.6 us (an
// empty graph takes 6).  A word for every token instead of a bit, cleared and read
// by 16 CTAs a row, took 60, and with the doubles inside the sweep, where a few
// lanes of almost every warp have one, 148.
#include <math.h>

#include <algorithm>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int kThreads = 512;
constexpr unsigned kMaxCtas = 16;  // of a row
constexpr int kSlots = 4096;       // marked tokens computed at a time
constexpr int kKeep = 8;           // history entries a thread keeps
constexpr int kStripe = 1024;      // consecutive tokens of one CTA
constexpr int kStripeBits = 10;
constexpr uint32_t kTopBit = 1u << 31;  // of `said`: the prompt has it

struct LogitsParams {
  const __nv_bfloat16* logits;
  int64_t ld;
  int64_t vocab;
  int chunk;  // tokens a CTA, a multiple of kStripe
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
B200_DEV Best warp_better(Best b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    b = better(b, Best{__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)});
  return b;
}

B200_DEV void cluster_store8(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Exclusive prefix sum of one value a thread; *total the sum of all.
B200_DEV int block_scan(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sums[w] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) {
    if (k < w) before += sums[k];
    all += sums[k];
  }
  *total = all;
  return before + inc - v;
}

// The larger of two bf16 pairs, NaN only where both are.
B200_DEV uint32_t max_pair(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
constexpr uint32_t kLowPair = 0xff80ff80u;  // -inf, -inf
// All ones in the halves whose bit of `two` is set.
B200_DEV uint32_t spread2(uint32_t two) { return (two & 1u) * 0xffffu | ((two >> 1) & 1u) * 0xffff0000u; }

struct Row {  // one row's lists
  const int32_t* history;
  int len, prompt;
  const int32_t* bias_ids;
  const float* bias_values;
  int biases;
};

// HIST / BIAS: the call has a history / a bias list.
template <bool HIST, bool BIAS>
__global__ void __launch_bounds__(kThreads, 2) logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ Best warp_best[kThreads / 32];
  __shared__ Best cta_best[kMaxCtas];  // the first CTA's: one of each CTA of the row
  __shared__ int sums[kThreads / 32];
  constexpr bool kLists = HIST || BIAS;
  constexpr int kAhead = 4;  // 16-byte loads in flight
  const int words = p.chunk / 32;
  uint32_t* marks = smem;                                     // [words]
  int* before = reinterpret_cast<int*>(marks + words);        // [words] marked tokens before each word
  int* token = before + words;                                // [kSlots] a marked token
  uint32_t* said = reinterpret_cast<uint32_t*>(token + kSlots);  // [kSlots] times behind the prompt | kTopBit
  uint32_t* lead = said + kSlots;                             // [kSlots] entries from its first bias to the list's end
  uint32_t* listed = lead + kSlots;                           // [kSlots] its biases
  pdl_trigger();
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // every CTA has started: waited for at the end
  const int64_t row = blockIdx.x / ctas;
  const int turn = __ffs(ctas) - 1;  // ctas is a power of two
  const int vocab = (int)p.vocab;
  const int tid = threadIdx.x;
  // token of this CTA's `at`, and the other way (-1: not this CTA's)
  auto token_of = [&](int at) { return ((((at >> kStripeBits) << turn) + rank) << kStripeBits) + (at & (kStripe - 1)); };
  auto place_of = [&](int id) {
    const int stripe = id >> kStripeBits;
    return (uint32_t)id < (uint32_t)vocab && (stripe & (ctas - 1)) == rank
               ? ((stripe >> turn) << kStripeBits) + (id & (kStripe - 1)) : -1;
  };
  const int nv = p.vec ? p.chunk / 8 : 0;  // groups of 8 tokens; some may lie behind the vocabulary
  if (kLists)
    for (int i = tid; i < words; i += kThreads) marks[i] = 0;
  pdl_wait();

  const __nv_bfloat16* in = p.logits + row * p.ld;
  __nv_bfloat16* out = p.out ? p.out + row * p.ldo : nullptr;
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int64_t m = p.mask_rows ? p.mask_rows[row] : row;
    if (m >= p.num_masks || m < -1) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
    } else if (m >= 0) {
      mask = p.mask + m * p.mask_ld;
    }
  }
  uint4 raw[kAhead];
  uint32_t bits[kAhead];  // the mask's words
  auto load = [&](int c0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (c0 + k * kThreads < nv) {
        const int id = token_of((c0 + k * kThreads) * 8);
        if (id + 8 <= vocab) {
          raw[k] = *reinterpret_cast<const uint4*>(in + id);
          bits[k] = mask ? mask[id >> 5] : 0xffffffffu;
        }
      }
  };
  load(tid);  // on their way while the lists are read
  Row r{};
  if (HIST) {
    r.history = p.history + row * p.history_ld;
    r.len = p.lens[row];
    r.prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
    if (r.len < 0 || r.len > p.history_ld || r.prompt < 0 || r.prompt > r.len) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
      r.len = (int)min((int64_t)max(r.len, 0), p.history_ld);
      r.prompt = min(max(r.prompt, 0), r.len);
    }
  }
  if (BIAS) {
    const int b0 = p.bias_offsets[row];
    r.biases = p.bias_offsets[row + 1] - b0;
    if (b0 < 0 || r.biases < 0) {
      if (tid == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
      r.biases = 0;
    }
    r.bias_ids = p.bias_ids + b0;
    r.bias_values = p.bias_values + b0;
  }

  // ---- which tokens are touched ----
  // The first entries of both lists stay in registers, all on their way at once.
  int32_t said_id[kKeep], bias_id;
  if (HIST)
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (tid + k * kThreads < r.len) said_id[k] = r.history[tid + k * kThreads];
  if (BIAS && tid < r.biases) bias_id = r.bias_ids[tid];
  int marked = 0;
  if (kLists) {
    __syncthreads();
    auto mark = [&](int32_t id) {
      const int at = place_of(id);
      if (at >= 0) atomicOr(&marks[at >> 5], 1u << (at & 31));
      else if ((uint32_t)id >= (uint32_t)vocab) raise_error(p.err, DEV_ERR_BAD_INDEX);
    };
    if (HIST) {
#pragma unroll
      for (int k = 0; k < kKeep; ++k)
        if (tid + k * kThreads < r.len) mark(said_id[k]);
      for (int i = tid + kKeep * kThreads; i < r.len; i += kThreads) mark(r.history[i]);
    }
    if (BIAS) {
      if (tid < r.biases) mark(bias_id);
      for (int i = tid + kThreads; i < r.biases; i += kThreads) mark(r.bias_ids[i]);
    }
    __syncthreads();
    const int per = (words + kThreads - 1) / kThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int mine = 0;
    for (int w = w0; w < w1; ++w) mine += __popc(marks[w]);
    int at = block_scan(mine, sums, &marked);
    for (int w = w0; w < w1; ++w) {
      before[w] = at;
      at += __popc(marks[w]);
    }
  }

  // ---- the sweep: copies, masks, the best of the untouched (bf16 values: compared as they are) ----
  float plain_v = -INFINITY;
  int plain_i = -1;
  for (int c0 = tid; c0 < nv; c0 += kAhead * kThreads) {
    if (c0 != tid) load(c0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = c0 + k * kThreads;
      if (c >= nv) break;
      const int id = token_of(c * 8);
      if (id + 8 > vocab) break;  // and all behind it
      uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
      uint32_t skip = kLists ? reinterpret_cast<const uint8_t*>(marks)[c] : 0;
      const uint32_t hidden = ~(bits[k] >> (id & 31)) & 0xffu;
      if (hidden) {
        skip |= hidden;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t h = spread2(hidden >> (2 * i));
          w[i] = (w[i] & ~h) | (kLowPair & h);
        }
      }
      if (out) *reinterpret_cast<uint4*>(out + id) = make_uint4(w[0], w[1], w[2], w[3]);
      if (skip) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t h = spread2(skip >> (2 * i));
          w[i] = (w[i] & ~h) | (kLowPair & h);
        }
      }
      uint32_t top = max_pair(max_pair(w[0], w[1]), max_pair(w[2], w[3]));
      const float most = fmaxf(__uint_as_float(top << 16), __uint_as_float(top & 0xffff0000u));
      if (most > plain_v) {  // seldom, after the first few
        plain_v = most;
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (__uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) == most) plain_i = id + i;
      }
    }
  }
  // rows that 16-byte accesses do not fit, and the last few tokens of those that they do
  int rest = 0;
  if (p.vec) rest = vocab % 8 != 0 && place_of(vocab & ~7) >= 0 ? place_of(vocab & ~7) : p.chunk;
  for (int at = rest + tid; at < p.chunk; at += kThreads) {
    const int id = token_of(at);
    if (id >= vocab) break;
    __nv_bfloat16 v = in[id];
    const float x = bf2f(v);
    if (mask && !((mask[id >> 5] >> (id & 31)) & 1u)) {
      v = __float2bfloat16_rn(-INFINITY);
    } else if (!(kLists && ((marks[at >> 5] >> (at & 31)) & 1u)) && x > plain_v) {
      plain_v = x;
      plain_i = id;
    }
    if (out) out[id] = v;
  }
  Best best{(double)plain_v, plain_i < 0 ? INT64_MAX : plain_i};

  // ---- the touched tokens, kSlots at a time ----
  if (kLists && marked > 0) {
    const bool rep = HIST && p.repetition, frq = HIST && p.frequency, prs = HIST && p.presence;
    const double repetition = rep ? (double)p.repetition[row] : 1.0;
    const double frequency = frq ? (double)p.frequency[row] : 0.0;
    const double presence = prs ? (double)p.presence[row] : 0.0;
    for (int s0 = 0; s0 < marked; s0 += kSlots) {
      const int slots = min(kSlots, marked - s0);
      __syncthreads();  // `before` is written; the last turn's slots are read, and the sweep's stores are done
      for (int i = tid; i < slots; i += kThreads) said[i] = lead[i] = listed[i] = 0;
      __syncthreads();
      // the slot of a token of this part, or -1
      auto slot_of = [&](int32_t id) -> int {
        const int at = place_of(id);
        if (at < 0) return -1;
        const int s = before[at >> 5] + __popc(marks[at >> 5] & ((1u << (at & 31)) - 1)) - s0;
        if (s < 0 || s >= slots) return -1;
        token[s] = id;
        return s;
      };
      auto say = [&](int i, int32_t id) {
        const int s = slot_of(id);
        if (s < 0) return;
        if (i < r.prompt) atomicOr(&said[s], kTopBit);
        else atomicAdd(&said[s], 1u);
      };
      // a token's first entry leads: it is worth the most counted from the end
      auto list = [&](int i, int32_t id) {
        const int s = slot_of(id);
        if (s < 0) return;
        atomicMax(&lead[s], (uint32_t)(r.biases - i));
        atomicAdd(&listed[s], 1u);
      };
      if (HIST) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
          if (tid + k * kThreads < r.len) say(tid + k * kThreads, said_id[k]);
        for (int i = tid + kKeep * kThreads; i < r.len; i += kThreads) say(i, r.history[i]);
      }
      if (BIAS) {
        if (tid < r.biases) list(tid, bias_id);
        for (int i = tid + kThreads; i < r.biases; i += kThreads) list(i, r.bias_ids[i]);
      }
      __syncthreads();
      for (int base = tid & ~31; base < slots; base += kThreads) {
        const int s = base + (tid & 31);
        const int id = s < slots ? token[s] : 0;
        const bool mine = s < slots && !(mask && !((mask[id >> 5] >> (id & 31)) & 1u));
        double v = mine ? (double)bf2f(in[id]) : 0;
        const uint32_t w = HIST && mine ? said[s] : 0, l = BIAS && mine ? lead[s] : 0;
        if (w) {
          if (rep) v = v > 0 ? __ddiv_rn(v, repetition) : __dmul_rn(v, repetition);
          const uint32_t times = w & ~kTopBit;
          if (frq) v = __dsub_rn(v, __dmul_rn(frequency, (double)times));
          if (prs && times) v = __dsub_rn(v, presence);
        }
        if (BIAS) {
          const int first = r.biases - (int)l;
          double sum = l ? (double)r.bias_values[first] : 0;
          // tokens listed more than once: the warp looks through the list for one after the other, and adds in its order
          uint32_t many = __ballot_sync(0xffffffffu, l && listed[s] > 1);
          for (; many; many &= many - 1) {
            const int owner = __ffs(many) - 1;
            const int its = __shfl_sync(0xffffffffu, id, owner);
            for (int e0 = __shfl_sync(0xffffffffu, first, owner) + 1; e0 < r.biases; e0 += 32) {
              const int e = e0 + (tid & 31);
              const bool same = e < r.biases && r.bias_ids[e] == its;
              const float value = same ? r.bias_values[e] : 0.f;
              for (uint32_t hits = __ballot_sync(0xffffffffu, same); hits; hits &= hits - 1) {
                const double add = (double)__shfl_sync(0xffffffffu, value, __ffs(hits) - 1);
                if ((tid & 31) == owner) sum = __dadd_rn(sum, add);
              }
            }
          }
          if (l) v = __dadd_rn(v, sum);
        }
        if (!mine) continue;
        if (v > best.v || (v == best.v && v > -INFINITY && id < best.i)) best = {v, id};
        if (out) out[id] = __double2bfloat16(v);
      }
    }
  }

  // ---- the greedy token: the CTAs' bests meet in the first one's shared memory ----
  if (p.next) {
    best = warp_better(best);
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) best = warp_better(tid < kThreads / 32 ? warp_best[tid] : Best{-INFINITY, INT64_MAX});
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (p.next && tid == 0) {
    const uint32_t at = cluster_map(smem_u32(&cta_best[rank]), 0);
    cluster_store8(at, (uint64_t)__double_as_longlong(best.v));
    cluster_store8(at + 8, (uint64_t)best.i);
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (p.next && rank == 0 && tid < 32) {
    best = warp_better(tid < ctas ? cta_best[tid] : Best{-INFINITY, INT64_MAX});
    if (tid == 0) p.next[row] = best.i == INT64_MAX ? -1 : best.i;
  }
}

// Shared memory of a part: a bit and an eighth of a count a token, and the slots.
int64_t part_bytes(int64_t chunk) { return chunk / 32 * 8 + kSlots * 16; }
constexpr int64_t kMaxSmem = 224 * 1024;

template <bool HIST, bool BIAS>
int launch(const LogitsParams& p, int64_t rows, unsigned ctas, cudaStream_t stream) {
  auto k = logits_kernel<HIST, BIAS>;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERROR_UNSUPPORTED;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem) != cudaSuccess ||
        cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess ||
        cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    done[dev] = true;
  }
  const size_t smem = HIST || BIAS ? (size_t)part_bytes(p.chunk) : 0;
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
  if (rows > INT32_MAX / 16 || vocab > (1 << 23) || history_ld > (1 << 30)) return B200_ERROR_UNSUPPORTED;
  if (rows == 0) return B200_OK;

  // CTAs of a row: as many as run at once (two an SM), at most 16, each with
  // 1024 tokens or more.
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  unsigned ctas = 1;
  while (ctas < kMaxCtas && (int64_t)ctas * 1024 < vocab && rows * ctas * 2 <= 2 * sms) ctas *= 2;
  const int64_t stripes = (vocab + kStripe - 1) / kStripe;
  auto part = [&](unsigned c) { return (stripes + c - 1) / c * kStripe; };
  while (ctas < kMaxCtas && part_bytes(part(ctas)) > kMaxSmem) ctas *= 2;
  const int64_t chunk = part(ctas);
  if (part_bytes(chunk) > kMaxSmem) return B200_ERROR_UNSUPPORTED;
  const int vec = (pl & 15u) == 0 && ld % 8 == 0 && (!out || ((po & 15u) == 0 && ldo % 8 == 0));
  const LogitsParams p{static_cast<const __nv_bfloat16*>(logits), ld, vocab, (int)chunk, history, history_ld,
                       prompt_lens, lens, repetition, frequency, presence, bias_offsets, bias_ids, bias_values, mask,
                       mask_ld, num_masks, mask_rows, static_cast<__nv_bfloat16*>(out), ldo, next, vec,
                       b200::error_word(dev)};
  if (hist) return bias ? launch<true, true>(p, rows, ctas, stream) : launch<true, false>(p, rows, ctas, stream);
  return bias ? launch<false, true>(p, rows, ctas, stream) : launch<false, false>(p, rows, ctas, stream);
}

// Block tables and slot maps of a paged KV cache from request lengths.
//
// extend:  with blocks(x) = ceil(x / block_size), sequence i needs
//   need_i = blocks(cached_i + new_i) - blocks(cached_i) further blocks.  The
//   j-th of them is free_blocks[count - 1 - (need_0 + .. + need_(i-1)) - j]:
//   the free list is a stack, served in sequence order, so the tables follow
//   from the lengths alone.  Token t of the step lies at position
//   cached_i + (t - cu_i) and in slot table[i, p / bs] * bs + p % bs.
// release: the blocks between blocks(min(cached_i, keep_i)) and
//   blocks(cached_i) go on top of the stack, in sequence and block order.
//
// Both are prefix sums over the sequences and then a gather an output: a few
// bytes a token, so what bounds them is the start of a launch and two dependent
// trips to memory.  One cluster of up to 16 CTAs runs a call: every CTA sums all
// sequences by itself (8192 lengths are 64 KB from L2, cheaper than handing
// sums over), the cluster meets once so that outputs may lie where inputs lay,
// and the CTAs share the entries and tokens.  A cluster instead of a grid
// because of that meeting: without it a step could not update its lengths and
// its free count in place, which a replayed graph needs.  104 thousand tokens of
// 2048 sequences take 16.4 us in a replayed graph with L2 flushed (an empty one
// takes 6); one token at a time in 8 CTAs, strided over all of them, they took 34.8.
#include <algorithm>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxSeqs = 8192;
constexpr int kAtOnce = 4;
constexpr unsigned kMaxCtas = 16;
constexpr int kPerThread = kMaxSeqs / kThreads;

B200_DEV int64_t warp_scan(int64_t v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Exclusive block-wide prefix sums of two values a thread; totals of both.  scratch: 2 * 33 values.
B200_DEV void block_scan2(int64_t& a, int64_t& b, int64_t* scratch, int64_t& total_a, int64_t& total_b) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t ia = warp_scan(a), ib = warp_scan(b);
  if (lane == 31) {
    scratch[w] = ia;
    scratch[33 + w] = ib;
  }
  __syncthreads();
  if (w == 0) {
    const int64_t va = scratch[lane], vb = scratch[33 + lane];
    const int64_t sa = warp_scan(va), sb = warp_scan(vb);
    scratch[lane] = sa - va;
    scratch[33 + lane] = sb - vb;
    if (lane == 31) {
      scratch[32] = sa;
      scratch[65] = sb;
    }
  }
  __syncthreads();
  a = scratch[w] + ia - a;
  b = scratch[33 + w] + ib - b;
  total_a = scratch[32];
  total_b = scratch[65];
  __syncthreads();
}

// The sequence i >= at with sums[i] <= x < sums[i + 1] (sums ascending,
// sums[at] <= x < sums[n]): steps that double from `at`, then halving.  Items
// are walked in ascending order, so most calls end at the first comparison.
B200_DEV int find(const int* sums, int n, int at, int x) {
  if (x < sums[at + 1]) return at;
  int lo = at + 1, step = 1;  // sums[lo] <= x
  while (lo + step < n && sums[lo + step] <= x) {
    lo += step;
    step <<= 1;
  }
  int hi = min(lo + step, n);  // x < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Division by the block size: a shift where it is a power of two.
struct BlockSize {
  int bs, shift;
  explicit BlockSize(int size) : bs(size), shift((size & (size - 1)) == 0 ? __builtin_ctz((unsigned)size) : -1) {}
  B200_DEV int quotient(int x) const { return shift >= 0 ? x >> shift : x / bs; }
};
// Blocks of `tokens` (at most INT32_MAX, and a sum with bs - 1 fits 32 unsigned bits).
B200_DEV int blocks_of(int tokens, const BlockSize& s) {
  const uint32_t up = (uint32_t)tokens + (uint32_t)(s.bs - 1);
  return (int)(s.shift >= 0 ? up >> s.shift : up / (uint32_t)s.bs);
}

struct Lens {
  int* cached;  // tokens each sequence holds
  int* tokens;  // [n + 1] prefix sums of new tokens (extend)
  int* blocks;  // [n + 1] prefix sums of blocks taken or given back
};

B200_DEV Lens carve(uint8_t* smem, int n) {
  Lens l;
  l.cached = reinterpret_cast<int*>(smem);
  l.tokens = l.cached + n;
  l.blocks = l.tokens + n + 1;
  return l;
}

// Reads both length arrays of the call into shared memory as sums.  EXTEND: second = new tokens, a sequence takes
// blocks; else second = tokens to keep, it gives blocks back.  Returns false when a length is out of range.
template <bool EXTEND>
B200_DEV bool read_lengths(const int32_t* cached, const int32_t* second, int n, const BlockSize& bs, int64_t room, Lens l,
                           int64_t* scratch, int64_t& total_tokens, int64_t& total_blocks) {
  const int per = (n + kThreads - 1) / kThreads;  // <= kPerThread consecutive sequences a thread
  const int first = threadIdx.x * per;
  int tok[kPerThread], blk[kPerThread];
  int64_t st = 0, sb = 0;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    tok[k] = blk[k] = 0;
    const int i = first + k;
    if (k < per && i < n) {
      int64_t c = cached[i], s = second[i];
      if (c < 0 || s < 0 || (EXTEND ? c + s : c) > room) {
        bad = true;
        c = s = 0;
      }
      l.cached[i] = (int)c;
      if (EXTEND) {
        tok[k] = (int)s;
        blk[k] = blocks_of((int)(c + s), bs) - blocks_of((int)c, bs);
      } else {
        tok[k] = (int)min(c, s);
        blk[k] = blocks_of((int)c, bs) - blocks_of(tok[k], bs);
      }
      st += tok[k];
      sb += blk[k];
    }
  }
  block_scan2(st, sb, scratch, total_tokens, total_blocks);
  bad = __syncthreads_or(bad);
  if (total_tokens > INT32_MAX || total_blocks > INT32_MAX) {
    if (EXTEND) bad = true;  // 32-bit sums would wrap (release keeps lengths, not sums, in `tokens`)
  }
  if (!bad) {
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = first + k;
      if (k < per && i < n) {
        l.tokens[i] = EXTEND ? (int)st : tok[k];
        l.blocks[i] = (int)sb;
        st += tok[k];
        sb += blk[k];
      }
    }
    if (threadIdx.x == 0) {
      if (EXTEND) l.tokens[n] = (int)total_tokens;
      l.blocks[n] = (int)total_blocks;
    }
  }
  __syncthreads();
  return !bad;
}

struct ExtendParams {
  const int32_t* cached;
  const int32_t* more;
  int n;
  BlockSize bs;
  int32_t* tables;
  int width;
  const int32_t* free_blocks;
  const int32_t* free_count;
  int64_t num_blocks;
  int32_t* context;
  int32_t* cu;
  int64_t* positions;
  int64_t* slots;
  int64_t capacity;
  int32_t* free_left;
  int32_t* missing;
  unsigned* err;
};

__global__ void __launch_bounds__(kThreads) extend_kernel(const ExtendParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t scratch[66];
  pdl_trigger();
  pdl_wait();
  const Lens l = carve(smem, p.n);
  const BlockSize bs = p.bs;
  const int rank = (int)cluster_rank(), ctas = (int)cluster_size();
  const int count = *p.free_count;
  int64_t tokens, need;
  const bool read = read_lengths<true>(p.cached, p.more, p.n, bs, (int64_t)p.width * bs.bs, l, scratch, tokens, need);
  const bool sane = read && count >= 0 && count <= p.num_blocks && tokens <= p.capacity;
  const bool fits = sane && need <= count;
  if (!sane && rank == 0 && threadIdx.x == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
  if (!read)  // the sums were not written; lengths are handed on as they were
    for (int i = threadIdx.x; i < p.n; i += kThreads) l.cached[i] = p.cached[i];
  cluster_sync();  // every CTA has read the lengths and the count: outputs may overwrite them
  if (rank == 0) {
    for (int i = threadIdx.x; i < p.n; i += kThreads) {
      p.context[i] = l.cached[i] + (fits ? l.tokens[i + 1] - l.tokens[i] : 0);
      if (p.cu) p.cu[i + 1] = fits ? l.tokens[i + 1] : 0;
    }
    if (threadIdx.x == 0) {
      if (p.cu) p.cu[0] = 0;
      *p.free_left = fits ? count - (int)need : count;
      if (p.missing) *p.missing = fits ? 0 : sane ? (int)(need - count) : -1;
    }
  }
  // A warp takes a run of entries, and of tokens, 32 side by side and kAtOnce of
  // those in a turn, so that as many loads from the tables are on their way
  // together and a lane's next item is mostly of the same sequence or the next.
  const int64_t warps = (int64_t)ctas * (kThreads / 32), warp = (int64_t)rank * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  auto run_of = [&](int64_t items) { return (items + warps * 32 - 1) / (warps * 32) * 32; };
  if (fits) {
    int i = 0;
    const int64_t run = run_of(need), end = min((warp + 1) * run, need);
    for (int64_t e0 = warp * run + lane; e0 < end; e0 += kAtOnce * 32) {
      int32_t b[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (e0 + k * 32 < end) b[k] = p.free_blocks[count - 1 - (e0 + k * 32)];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int64_t e = e0 + k * 32;
        if (e >= end) break;
        i = find(l.blocks, p.n, i, (int)e);
        if (b[k] < 0 || b[k] >= p.num_blocks) {
          raise_error(p.err, DEV_ERR_BAD_INDEX);
          b[k] = -1;
        }
        p.tables[(int64_t)i * p.width + blocks_of(l.cached[i], bs) + (int)e - l.blocks[i]] = b[k];
      }
    }
  }
  if (p.positions || p.slots) {
    int i = 0;
    const int64_t run = run_of(p.capacity), end = min((warp + 1) * run, p.capacity);
    for (int64_t t0 = warp * run + lane; t0 < end; t0 += kAtOnce * 32) {
      int at[kAtOnce];
      int32_t b[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int64_t t = t0 + k * 32;
        at[k] = -1;
        if (fits && t < tokens && t < end) {
          i = find(l.tokens, p.n, i, (int)t);
          at[k] = l.cached[i] + (int)t - l.tokens[i];
          const int col = bs.quotient(at[k]), held = blocks_of(l.cached[i], bs);
          b[k] = col < held ? p.tables[(int64_t)i * p.width + col]
                            : p.free_blocks[count - 1 - (l.blocks[i] + col - held)];
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int64_t t = t0 + k * 32;
        if (t >= end) break;
        int64_t slot = -1;
        if (at[k] >= 0) {
          if (b[k] >= 0 && b[k] < p.num_blocks) slot = (int64_t)b[k] * bs.bs + at[k] - bs.quotient(at[k]) * bs.bs;
          else raise_error(p.err, DEV_ERR_BAD_INDEX);
        }
        if (p.positions) p.positions[t] = max(at[k], 0);
        if (p.slots) p.slots[t] = slot;
      }
    }
  }
}

struct ReleaseParams {
  const int32_t* cached;
  const int32_t* keep;
  int n;
  BlockSize bs;
  const int32_t* tables;
  int width;
  int32_t* free_blocks;
  int64_t free_capacity;
  const int32_t* free_count;
  int64_t num_blocks;
  int32_t* lens;
  int32_t* free_left;
  unsigned* err;
};

__global__ void __launch_bounds__(kThreads) release_kernel(const ReleaseParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t scratch[66];
  pdl_trigger();
  pdl_wait();
  const Lens l = carve(smem, p.n);
  const BlockSize bs = p.bs;
  const int rank = (int)cluster_rank(), ctas = (int)cluster_size();
  const int count = *p.free_count;
  int64_t kept, drop;
  const bool read = read_lengths<false>(p.cached, p.keep, p.n, bs, (int64_t)p.width * bs.bs, l, scratch, kept, drop);
  const bool fits = read && count >= 0 && count + drop <= p.free_capacity;
  if (!fits && rank == 0 && threadIdx.x == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
  if (!read)
    for (int i = threadIdx.x; i < p.n; i += kThreads) l.cached[i] = p.cached[i];
  cluster_sync();  // as above
  if (rank == 0) {
    for (int i = threadIdx.x; i < p.n; i += kThreads) p.lens[i] = fits ? l.tokens[i] : l.cached[i];
    if (threadIdx.x == 0) *p.free_left = fits ? count + (int)drop : count;
  }
  if (!fits) return;
  int i = 0;
  for (int64_t e = (int64_t)rank * kThreads + threadIdx.x; e < drop; e += (int64_t)ctas * kThreads) {
    i = find(l.blocks, p.n, i, (int)e);
    const int32_t b = p.tables[(int64_t)i * p.width + blocks_of(l.tokens[i], bs) + (int)e - l.blocks[i]];
    if (b < 0 || b >= p.num_blocks) raise_error(p.err, DEV_ERR_BAD_INDEX);  // handed on; extend refuses it
    p.free_blocks[count + e] = b;
  }
}

int smem_bytes(int n) { return (3 * n + 2) * (int)sizeof(int); }

// Opt a kernel into the shared memory of kMaxSeqs sequences, once per device.
template <auto Kernel>
bool allow_smem() {
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return false;
  if (!done[dev])
    done[dev] = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kMaxSeqs)) ==
                    cudaSuccess &&
                cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
  return done[dev];
}

// CTAs of the cluster: one for each 1024 items (tokens or table entries), at most 16.
unsigned cluster_for(int64_t items) {
  unsigned c = 1;
  while (c < kMaxCtas && (int64_t)c * kThreads < items) c *= 2;
  return c;
}

bool al4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool al8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

unsigned* this_error_word() {
  int dev = 0;
  cudaGetDevice(&dev);
  return b200::error_word(dev);
}

}  // namespace

extern "C" int b200_block_tables_extend(const int32_t* cached_lens, const int32_t* new_lens, int num_seqs,
                                        int block_size, int32_t* block_tables, int max_blocks_per_seq,
                                        const int32_t* free_blocks, const int32_t* free_count, int64_t num_blocks,
                                        int32_t* context_lens, int32_t* cu_seqlens, int64_t* positions,
                                        int64_t* slots, int64_t capacity, int32_t* free_left, int32_t* missing,
                                        b200_stream_t stream) {
  if ((num_seqs > 0 && (!cached_lens || !new_lens || !block_tables || !context_lens)) || !free_blocks || !free_count ||
      !free_left || num_seqs < 0 || block_size <= 0 || max_blocks_per_seq <= 0 || num_blocks <= 0 || capacity < 0)
    return B200_ERROR_INVALID_PARAM;
  for (const void* q : {(const void*)cached_lens, (const void*)new_lens, (const void*)block_tables,
                        (const void*)free_blocks, (const void*)free_count, (const void*)context_lens,
                        (const void*)cu_seqlens, (const void*)free_left, (const void*)missing})
    if (!al4(q)) return B200_ERROR_INVALID_PARAM;
  if (!al8(positions) || !al8(slots)) return B200_ERROR_INVALID_PARAM;
  if (num_seqs > kMaxSeqs || num_blocks > INT32_MAX || capacity > INT32_MAX ||
      (int64_t)max_blocks_per_seq * block_size > INT32_MAX)
    return B200_ERROR_UNSUPPORTED;
  if (!allow_smem<extend_kernel>()) return B200_ERROR_UNSUPPORTED;
  const ExtendParams p{cached_lens,  new_lens, num_seqs,  BlockSize(block_size), block_tables, max_blocks_per_seq,
                       free_blocks,  free_count, num_blocks, context_lens, cu_seqlens, positions,
                       slots,        capacity,   free_left,  missing,      this_error_word()};
  const unsigned c = cluster_for(std::max<int64_t>(num_seqs, capacity));
  launch_clusters(extend_kernel, c, dim3(c), kThreads, smem_bytes(num_seqs), stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

extern "C" int b200_block_tables_release(const int32_t* cached_lens, const int32_t* keep_lens, int num_seqs,
                                         int block_size, const int32_t* block_tables, int max_blocks_per_seq,
                                         int32_t* free_blocks, int64_t free_capacity, const int32_t* free_count,
                                         int64_t num_blocks, int32_t* lens, int32_t* free_left,
                                         b200_stream_t stream) {
  if ((num_seqs > 0 && (!cached_lens || !keep_lens || !block_tables || !lens)) || !free_blocks || !free_count ||
      !free_left || num_seqs < 0 || block_size <= 0 || max_blocks_per_seq <= 0 || num_blocks <= 0 || free_capacity < 0)
    return B200_ERROR_INVALID_PARAM;
  for (const void* q : {(const void*)cached_lens, (const void*)keep_lens, (const void*)block_tables,
                        (const void*)free_blocks, (const void*)free_count, (const void*)lens, (const void*)free_left})
    if (!al4(q)) return B200_ERROR_INVALID_PARAM;
  if (num_seqs > kMaxSeqs || num_blocks > INT32_MAX || free_capacity > INT32_MAX ||
      (int64_t)max_blocks_per_seq * block_size > INT32_MAX)
    return B200_ERROR_UNSUPPORTED;
  if (!allow_smem<release_kernel>()) return B200_ERROR_UNSUPPORTED;
  const ReleaseParams p{cached_lens, keep_lens,  num_seqs,   BlockSize(block_size), block_tables, max_blocks_per_seq, free_blocks,
                        free_capacity, free_count, num_blocks, lens,       free_left,    this_error_word()};
  const unsigned c = cluster_for((int64_t)num_seqs * std::min(max_blocks_per_seq, 8));
  launch_clusters(release_kernel, c, dim3(c), kThreads, smem_bytes(num_seqs), stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

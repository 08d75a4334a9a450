// The parts of a shared prefix's attention, as the kernel that computes them
// (shared_prefix.cu) leaves them and the one that joins them with each
// sequence's own tokens (paged_window.cu) reads them.
//
// Query rows are the batch's heads of one kv head: per_tile sequences of
// `group` heads fill a 128-row tile.  An item is a kv head and two row tiles
// (the last may be alone); its prefix has K = ceil(length / 128) key tiles.  The items' key tiles in a row,
// U of them, are dealt to W = min(workers, U) CTAs in stretches of U / W or one
// more (the first U mod W), so each has a tile at least.  Each stretch of
// an item is a part; the part of worker c in item i lies in slots 2 (c + i) and
// 2 (c + i) + 1, a row tile each: of two consecutive parts the later has a larger
// worker or item.
#pragma once

#include "common.cuh"

namespace b200 {

struct PrefixParts {
  float* parts;  // [slots][128][head_dim] outputs over their sums
  float* lse;    // [slots][128] log2 of the sums, with their maximum; -inf: no key has weight
  const int32_t* length;
  int max_length;
  int workers, row_tiles, per_tile, group;
};

B200_DEV int prefix_pairs(const PrefixParts& p) { return (p.row_tiles + 1) / 2; }
B200_DEV int prefix_length(const PrefixParts& p) { return max(0, min(*p.length, p.max_length)); }

// The stretches of U units: how many, the first unit of stretch c, the stretch of unit u.
struct PrefixDeal {
  int W, each, longer;  // the first `longer` stretches have each + 1 units
  B200_DEV PrefixDeal(const PrefixParts& p, int units) {
    W = max(1, min(p.workers, units));
    each = units / W;
    longer = units - each * W;
  }
  B200_DEV int first_unit(int c) const { return c * each + min(c, longer); }
  B200_DEV int worker(int u) const {
    const int cut = longer * (each + 1);
    return u < cut ? u / (each + 1) : longer + (u - cut) / each;
  }
};

// The parts of one sequence's heads [first_head, ..) of a kv head; a part's next is 256 rows on.
struct PrefixSpan {
  const float* parts = nullptr;
  const float* lse = nullptr;
  int count = 0;
};

B200_DEV PrefixSpan prefix_span(const PrefixParts& p, int sequence, int kv_head, int nkv, int first_head, int head_dim) {
  PrefixSpan s;
  const int K = (prefix_length(p) + 127) / 128;
  if (K == 0) return s;
  const int tile = sequence / p.per_tile, item = kv_head * prefix_pairs(p) + tile / 2;
  const PrefixDeal deal(p, K * nkv * prefix_pairs(p));
  const int w0 = deal.worker(item * K), w1 = deal.worker(item * K + K - 1);
  const int64_t row = (int64_t)(2 * (w0 + item) + tile % 2) * 128 + (sequence % p.per_tile) * p.group + first_head;
  s.count = w1 - w0 + 1;
  s.parts = p.parts + row * head_dim;
  s.lse = p.lse + row;
  return s;
}

// Single-token attention over the sequences' own tokens (paged_window.cu), joined with a prefix's parts when there are
// any (prefix.parts, of the kernel launched just before).  Arguments are checked by the callers.
int paged_window_launch(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                        const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
                        int nq, int nkv, int head_dim, int block_size, int64_t num_blocks, float scale, int window,
                        int sinks, void* out, int64_t out_stride, int max_context, const PrefixParts& prefix,
                        cudaStream_t stream);

// The checks that both entry points make of their common arguments (a status, B200_OK to go on).
int paged_window_check(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                       const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
                       int nq, int nkv, int head_dim, int block_size, int64_t num_blocks, float scale, const void* out,
                       int64_t out_stride, int max_context);

}  // namespace b200

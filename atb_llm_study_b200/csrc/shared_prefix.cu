// Single-token attention of a batch whose sequences share a long prefix, the
// prefix computed once for all.
//
//   out = (2^(lse_0 - M) o_0 + sum_i 2^(lse_i - M) o_i) / (the weights' sum)
//
// with o_0 the attention over the sequence's own tokens, o_i over stretches of
// the prefix and lse their log2 sums: softmax over both is the sum of the parts
// weighted by their share of the whole sum.
//
// One token a sequence reads the cache once for 4 flops a byte and head, and a
// prefix in every sequence's table is read batch times.  Taken together, the
// batch's query heads of a kv head are the rows of a matrix product: the prefix
// is read once, and with 64 sequences of 4 heads a kv head the operations (256
// a byte) reach the tensor cores' rate at the time that the bytes take.  So
// this half runs on tcgen05 (tc_items.cuh), 128 rows a tile, the items' key
// tiles dealt evenly over the SMs, each stretch leaving a part in 32 bits; the
// kernel for the sequences' own tokens joins them (paged_window.cu), two
// launches in all.
//
// Measured, 64 sequences behind 16384 tokens with up to 1024 of their own, 32 / 8
// heads of 128: 67 us (floor 30, of which 20 for the own tokens); of 64: 45 (15).
// The prefix's share of the 67 is 25: 5 until the first scores (cold lengths, tables
// and tiles one after the other), 7 key tiles of two row tiles at 4200 cycles, and 2 a
// side for 64 KB of outputs.  Fewer CTAs, to let the other kernel run beside this one,
// gained nothing: its CTAs wait for these parts in their places.
#include <algorithm>

#include "shared_prefix.h"
#include "tc_items.cuh"

using namespace b200;

namespace {

template <int HD>
struct Prefix {
  static constexpr int HDK = HD, HDV = HD;
  using Cf = ItemsCfg<Prefix>;
  PrefixParts at;
  const int32_t* blocks;
  int64_t num_blocks;
  int nkv, block_size, batch;
  float scale_log2;

  struct Item {
    int n;       // key tiles of this stretch
    bool both;   // two row tiles
    int first;   // the first key tile
    int length;  // of the prefix
    int kvh, row_tile, slot;  // side 0's; side 1's follow
  };

  struct Cursor {
    const Prefix& p;
    int length;
    int K, unit, end;
    B200_DEV explicit Cursor(const Prefix& q) : p(q) {
      length = prefix_length(p.at);
      K = (length + kTile - 1) / kTile;
      const PrefixDeal deal(p.at, K * p.nkv * prefix_pairs(p.at));
      const bool has = K > 0 && (int)blockIdx.x < deal.W;
      unit = has ? deal.first_unit(blockIdx.x) : 0;
      end = has ? deal.first_unit(blockIdx.x + 1) : 0;
    }
    B200_DEV bool next(Item& it, unsigned*) {
      if (unit >= end) return false;
      const int item = unit / K, pairs = prefix_pairs(p.at);
      it.first = unit - item * K;
      it.n = min(end - unit, K - it.first);
      it.length = length;
      it.kvh = item / pairs;
      it.row_tile = item % pairs * 2;
      it.both = it.row_tile + 1 < p.at.row_tiles;
      it.slot = ((int)blockIdx.x + item) * 2;
      unit += it.n;
      return true;
    }
  };

  B200_DEV static int key0(const Item& it, int j) { return (it.first + j) * kTile; }
  B200_DEV static bool whole(const Item& it, int, int key) { return key + kTile <= it.length; }
  B200_DEV static uint32_t visible(const Item& it, int, int, int key) { return bit_range(0, it.length - key); }
  // box rows are the group's heads of per_tile sequences; rows behind them are not written, and not used
  B200_DEV static void load_q(const Prefix& p, const Item& it, int s, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar) {
    mbar_arrive_expect_tx(bar, Cf::BOXES_QK * p.at.per_tile * p.at.group * 128);
    for (int x = 0; x < Cf::BOXES_QK; ++x)
      tma_load_3d(dst + x * kBoxBytes, map, bar, 64 * x, it.kvh * p.at.group, (it.row_tile + s) * p.at.per_tile);
  }
  // a tile is one block of 128 tokens or two of 64, of which the second may lie behind the prefix: it is not loaded,
  // and its keys are hidden like the rest of a last block
  B200_DEV static void load(const Prefix& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map,
                            uint64_t* bar, unsigned* err) {
    const int key = key0(it, j), per = kTile / p.block_size;
    const int n = min(per, (it.length - key + p.block_size - 1) / p.block_size);
    mbar_arrive_expect_tx(bar, n * Cf::BOXES_QK * p.block_size * 128);
    for (int i = 0; i < n; ++i) {
      int blk = p.blocks[key / p.block_size + i];
      if (blk < 0 || blk >= p.num_blocks) {
        raise_error(err, DEV_ERR_BAD_INDEX);
        blk = 0;
      }
      const int row = (blk * p.nkv + it.kvh) * p.block_size;
      for (int x = 0; x < Cf::BOXES_QK; ++x)
        tma_load_2d(dst + x * kBoxBytes + i * p.block_size * 128, map, bar, 64 * x, row);
    }
  }
  B200_DEV static void load_k(const Prefix& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar, unsigned* err) {
    load(p, it, j, dst, map, bar, err);
  }
  B200_DEV static void load_v(const Prefix& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar, unsigned* err) {
    load(p, it, j, dst, map, bar, err);
  }
  B200_DEV static void store(const Prefix& p, const Item& it, int s, int row, float m, float l, uint32_t tO) {
    const int seqs = min(p.at.per_tile, p.batch - (it.row_tile + s) * p.at.per_tile);
    const bool valid = row < seqs * p.at.group;
    // Every row sees the stretch's keys, but where all its scores are -inf they have no weight beside other parts': the
    // part is zeros with a log sum of -inf.  (l is then what the polynomial leaves of 2^-126, or NaN where a score is.)
    const bool none = m == -INFINITY && l == l;
    const float inv = none ? 0.f : 1.f / l;
    float* o = p.at.parts + ((int64_t)(it.slot + s) * kTile + row) * HD;
    if (valid) p.at.lse[(int64_t)(it.slot + s) * kTile + row] = none ? -INFINITY : m + log2f(l);
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tO + c * 32, r);
      tmem_ld_wait();
      if (valid) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          Words8 w;
#pragma unroll
          for (int i = 0; i < 8; ++i) w.w[i] = __float_as_uint(__uint_as_float(r[8 * k + i]) * inv);
          store_32(o + c * 32 + k * 8, w);
        }
      }
    }
  }
};

struct Plan {
  int per_tile, row_tiles, workers;
  int64_t units, slots;
};

// SMs share the key tiles evenly, with no CTA left without one.  A part has two tiles of 128 rows.
Plan prefix_plan(int batch, int nq, int nkv, int max_prefix) {
  Plan p;
  p.per_tile = kTile / (nq / nkv);
  p.row_tiles = (batch + p.per_tile - 1) / p.per_tile;
  const int64_t items = (int64_t)nkv * ((p.row_tiles + 1) / 2);
  p.units = items * ((max_prefix + (int64_t)kTile - 1) / kTile);
  p.workers = (int)std::max<int64_t>(1, std::min<int64_t>(p.units, sm_count()));
  p.slots = 2 * (p.workers + items);
  return p;
}

int64_t plan_bytes(const Plan& p, int head_dim) { return p.slots * kTile * (head_dim + 1) * (int64_t)sizeof(float); }

template <int HD>
int launch_prefix(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int nq,
                  const Prefix<HD>& p, int64_t rows, cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  if (!encode_tiled_3d(&mq, q, HD, nq, p.batch, HD * 2, q_stride * 2, 64, p.at.group, p.at.per_tile) ||
      !encode_tiled_2d(&mk, k_cache, HD, rows, HD * 2, 64, p.block_size) ||
      !encode_tiled_2d(&mv, v_cache, HD, rows, HD * 2, 64, p.block_size))
    return B200_ERROR_UNSUPPORTED;
  return launch_items(mq, mk, mv, p, p.at.workers, stream);
}

}  // namespace

extern "C" int64_t b200_paged_decode_shared_workspace_bytes(int batch, int nq, int nkv, int head_dim, int max_prefix) {
  if (batch <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > kTile || (head_dim != 64 && head_dim != 128) ||
      max_prefix <= 0)
    return 0;
  return plan_bytes(prefix_plan(batch, nq, nkv, max_prefix), head_dim);
}

extern "C" int b200_paged_decode_shared(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                                        const int32_t* prefix_blocks, const int32_t* prefix_len, int max_prefix,
                                        const int32_t* block_tables, int max_blocks_per_seq,
                                        const int32_t* context_lens, int max_context, int batch, int nq, int nkv,
                                        int head_dim, int block_size, int64_t num_blocks, float scale, void* out,
                                        int64_t out_stride, void* workspace, int64_t workspace_bytes,
                                        b200_stream_t stream) {
  const int rc = paged_window_check(q, q_stride, k_cache, v_cache, block_tables, max_blocks_per_seq, context_lens,
                                    batch, nq, nkv, head_dim, block_size, num_blocks, scale, out, out_stride,
                                    max_context);
  if (rc != B200_OK) return rc;
  if (max_prefix < 0 || (max_prefix > 0 && (!prefix_blocks || !prefix_len)) ||
      (reinterpret_cast<uintptr_t>(prefix_blocks) & 3u) || (reinterpret_cast<uintptr_t>(prefix_len) & 3u))
    return B200_ERROR_INVALID_PARAM;
  if (nq / nkv > kTile || max_prefix > INT32_MAX - 256) return B200_ERROR_UNSUPPORTED;
  if (batch == 0) return B200_OK;
  PrefixParts at{};
  if (max_prefix > 0) {
    const Plan plan = prefix_plan(batch, nq, nkv, max_prefix);
    if (plan.units > INT32_MAX) return B200_ERROR_UNSUPPORTED;
    if (!workspace || workspace_bytes < plan_bytes(plan, head_dim) || (reinterpret_cast<uintptr_t>(workspace) & 31u))
      return B200_ERROR_INVALID_PARAM;
    at.parts = static_cast<float*>(workspace);
    at.lse = at.parts + plan.slots * kTile * head_dim;
    at.length = prefix_len;
    at.max_length = max_prefix;
    at.workers = plan.workers;
    at.row_tiles = plan.row_tiles;
    at.per_tile = plan.per_tile;
    at.group = nq / nkv;
    const int64_t rows = num_blocks * nkv * block_size;
    const float sl2 = scale * 1.4426950408889634f;
    const int r = head_dim == 128
                      ? launch_prefix<128>(q, q_stride, k_cache, v_cache, nq,
                                           Prefix<128>{at, prefix_blocks, num_blocks, nkv, block_size, batch, sl2},
                                           rows, stream)
                      : launch_prefix<64>(q, q_stride, k_cache, v_cache, nq,
                                          Prefix<64>{at, prefix_blocks, num_blocks, nkv, block_size, batch, sl2},
                                          rows, stream);
    if (r != B200_OK) return r;
  }
  // the sequences' own tokens: a window of all of them
  return paged_window_launch(q, q_stride, k_cache, v_cache, block_tables, max_blocks_per_seq, context_lens, batch, nq,
                             nkv, head_dim, block_size, num_blocks, scale, INT32_MAX, 0, out, out_stride, max_context,
                             at, stream);
}

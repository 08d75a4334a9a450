// Prompt attention with a sliding window and a few first tokens that stay
// visible: query i of a sequence sees keys j <= i with i - j < window or
// j < sinks.
//
// The tensor cores bound it: 4 flops a visible pair, head and dim, and a 128-row
// query tile touches window / 128 + 2 key tiles (the window's ends cut through
// one each) besides the sinks'.  Tiles without a visible pair are never
// loaded, so the time follows the window and not the prompt.  The two sides of an
// item (tc_items.cuh) are two heads that share their keys, or, where nq / nkv is
// odd, two query tiles of one head next to each other.  Items are walked with
// the heads of one sequence's rows side by side: those that share keys find them
// in L2.
//
// Measured, 32 / 8 heads of 128, replayed with pauses: 8 x 2048 with a window of
// 1024 in 281 us (736 TFLOP/s of visible pairs, 84 % of the pairs computed), 1 x
// 32768 with 4096 in 1.93 ms (1070 TFLOP/s, 65 % of the measured burst rate); back
// to back, under the power limit, 318 us and 2.23 ms.  A tile at the window's ends
// costs a side half as much again as a whole one.  The first of them with 16 / 8
// heads: 145 us, and 123 at 64, 119 at 32, 116 at 16 (narrow heads take the copies
// and products of 64-wide ones); 16 / 16 heads of 192 / 128 take 232 (556 TFLOP/s).
#include <algorithm>

#include "tc_items.cuh"

using namespace b200;

namespace {

// HEADS3D: heads narrower than the 64-column box, mapped as rows of their own (tc_attention.cuh)
template <int HDK_, int HDV_, bool HEADS3D>
struct Window {
  static constexpr int HDK = HDK_, HDV = HDV_;
  using Cf = ItemsCfg<Window>;
  __nv_bfloat16* out;
  int64_t os, ohs;
  const int32_t* cu;
  int nq, nkv, nseq, items, total, max_rows;
  int64_t qhs, khs, vhs;
  float scale_log2;
  int window, sinks, out_cols;
  bool pair_heads, by_tile;

  struct Item {
    int n;                       // key tiles
    bool both;                   // side 1 has rows
    int h0, h1, m0, m1;          // sides' heads and first query positions
    int kvh, start, len;         // len: the keys'
    int rows;                    // and the queries', up to max_seqlen
    int head, first;             // sink tiles, and the window's first tile
    int window, sinks;
    B200_DEV int at(int s) const { return s ? m1 : m0; }
    B200_DEV int head_of(int s) const { return s ? h1 : h0; }
  };

  // An item: two heads of a query tile, or two query tiles of a head, in one of two
  // orders.  By tile: the last tiles of all sequences first, which see most keys,
  // so that the walk ends with cheap items; it walks over numbers of sequences that
  // have no such tile.  By sequence: sequence s owns the numbers from
  // floor(cu[s] / rows) + s on, as many as it has tiles, or one more, whatever the
  // lengths, and the sequence of a number is found by halving.  By tile and by
  // sequence (us), at so many times the numbers of the other order: 8 x 2048 at 0.94
  // 271 and 294, at 1.12 246 and 239, at 1.24 222 and 218, at 1.39 198 and 182; 16 x
  // 1024 under a window of 256 at 1.22 139 and 142, at 1.62 109 and 104; 16 x 2048
  // with 8 / 8 heads at 1.08 120 and 127, at 1.22 115 and 114, at 1.62 95 and 82; 64
  // x 900 with 12 / 4 heads of 64 at 1.16 154 and 161, at 1.47 119 and 120.
  struct Cursor {
    const Window& p;
    int w;
    B200_DEV explicit Cursor(const Window& q) : p(q), w(blockIdx.x) {}
    B200_DEV bool next(Item& it, unsigned* err) {
      const int heads = p.pair_heads ? p.nq / 2 : p.nq, shift = p.pair_heads ? 7 : 8;
      for (; w < p.items; w += gridDim.x) {
        const int back = w / heads, h = w - back * heads;
        int lo = 0, m;  // sequence, tile
        if (p.by_tile) {
          m = p.items / heads / p.nseq - 1 - back / p.nseq;
          lo = back % p.nseq;
        } else {
          const int t = p.items / heads - 1 - back;
          for (int hi = p.nseq; hi - lo > 1;) {  // first number of lo <= t < first number of hi
            const int mid = (lo + hi) >> 1;
            if ((p.cu[mid] >> shift) + mid <= t) lo = mid;
            else hi = mid;
          }
          m = t - lo - (p.cu[lo] >> shift);
        }
        it.start = p.cu[lo];
        it.len = p.cu[lo + 1] - it.start;
        if (it.start < 0 || it.len > p.total - it.start) {  // rows outside the operands
          raise_error(err, DEV_ERR_BAD_INDEX);
          continue;
        }
        it.rows = min(it.len, p.max_rows);
        if (m < 0 || m > (it.rows - 1) >> shift) continue;
        const int m0 = m << shift;
        it.h0 = p.pair_heads ? 2 * h : h;
        it.h1 = p.pair_heads ? 2 * h + 1 : h;
        it.m0 = m0;
        it.m1 = p.pair_heads ? m0 : m0 + kTile;
        it.both = it.m1 < it.rows;
        it.kvh = it.h0 / (p.nq / p.nkv);
        it.first = max(0, m0 - p.window + 1) / kTile;
        it.head = min((p.sinks + kTile - 1) / kTile, it.first);
        it.n = it.head + (it.both ? it.m1 : m0) / kTile - it.first + 1;
        it.window = p.window;
        it.sinks = p.sinks;
        w += gridDim.x;
        return true;
      }
      return false;
    }
  };

  // The window's tiles from its second on, then its first, then the sinks': rows
  // meet their usual maximum at once, in a tile that they see as a whole, where
  // the few sinks or a window's first keys would give them one to outgrow.
  B200_DEV static int key0(const Item& it, int j) {
    const int rest = it.n - it.head - 1;
    return (j < rest ? it.first + 1 + j : j == rest ? it.first : j - rest - 1) * kTile;
  }
  B200_DEV static bool whole(const Item& it, int s, int key) {
    return key + kTile - 1 <= it.at(s) && key + kTile <= it.len &&
           (it.at(s) + kTile - 1 - key < it.window || key + kTile <= it.sinks);
  }
  // key <= i and key < len and (key > i - window or key < sinks), i the row's position
  B200_DEV static uint32_t visible(const Item& it, int s, int row, int key) {
    const int i = it.at(s) + row, end = min(i + 1, it.len) - key;
    return bit_range(i - it.window + 1 - key, end) | bit_range(0, min(it.sinks - key, end));
  }
  B200_DEV static void load_q(const Window& p, const Item& it, int s, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar) {
    mbar_arrive_expect_tx(bar, Cf::TILE_QK);
    if (HEADS3D) tma_load_3d(dst, map, bar, 0, it.head_of(s), it.start + it.at(s));
    else
      for (int x = 0; x < Cf::BOXES_QK; ++x)
        tma_load_2d(dst + x * kBoxBytes, map, bar, (int)(it.head_of(s) * p.qhs) + 64 * x, it.start + it.at(s));
  }
  B200_DEV static void load_k(const Window& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar, unsigned*) {
    mbar_arrive_expect_tx(bar, Cf::TILE_QK);
    if (HEADS3D) tma_load_3d(dst, map, bar, 0, it.kvh, it.start + key0(it, j));
    else
      for (int x = 0; x < Cf::BOXES_QK; ++x)
        tma_load_2d(dst + x * kBoxBytes, map, bar, (int)(it.kvh * p.khs) + 64 * x, it.start + key0(it, j));
  }
  B200_DEV static void load_v(const Window& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map,
                              uint64_t* bar, unsigned*) {
    mbar_arrive_expect_tx(bar, Cf::TILE_V);
    if (HEADS3D) tma_load_3d(dst, map, bar, 0, it.kvh, it.start + key0(it, j));
    else
      for (int x = 0; x < Cf::BOXES_V; ++x)
        tma_load_2d(dst + x * kBoxBytes, map, bar, (int)(it.kvh * p.vhs) + 64 * x, it.start + key0(it, j));
  }
  // O / l from TMEM as bf16 rows
  B200_DEV static void store(const Window& p, const Item& it, int s, int row, float m, float l, uint32_t tO) {
    const float inv = m == -INFINITY ? NAN : 1.f / l;  // every row sees itself: scores of -inf alone are 0 / 0
    const bool valid = it.at(s) + row < it.rows;
    __nv_bfloat16* o = p.out + (int64_t)(it.start + (valid ? it.at(s) + row : 0)) * p.os + (int64_t)it.head_of(s) * p.ohs;
#pragma unroll 1
    for (int c = 0; c < HDV / 32; ++c) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tO + c * 32, r);
      tmem_ld_wait();
      if (valid) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (HEADS3D && c * 32 + k * 8 >= p.out_cols) break;
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r[8 * k + i]) * inv;
          *reinterpret_cast<uint4*>(o + c * 32 + k * 8) = pack8(f);
        }
      }
    }
  }
};

}  // namespace

extern "C" int b200_flash_prefill_window(const void* q, int64_t q_stride, int64_t q_head_stride, const void* k,
                                         int64_t k_stride, int64_t k_head_stride, const void* v, int64_t v_stride,
                                         int64_t v_head_stride, void* out, int64_t out_stride,
                                         int64_t out_head_stride, const int32_t* cu_seqlens, int num_seqs,
                                         int max_seqlen, int64_t total_tokens, int nq, int nkv, int head_dim_qk,
                                         int head_dim_v, float scale, int window, int sinks, b200_stream_t stream) {
  if (!q || !k || !v || !out || !cu_seqlens || num_seqs < 0 || max_seqlen < 0 || total_tokens < 0 || nq <= 0 ||
      nkv <= 0 || nq % nkv || window <= 0 || sinks < 0 || !(scale > 0.f && scale < INFINITY))
    return B200_ERROR_INVALID_PARAM;
  const int hd = head_dim_qk, hdv = head_dim_v;
  if (!((hd == hdv && (hd == 128 || hd == 64 || hd == 32 || hd == 16)) || (hd == 192 && hdv == 128)))
    return B200_ERROR_UNSUPPORTED;
  for (int64_t s : {q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride, out_stride,
                    out_head_stride})
    if (s < 0 || s % 8 || s > INT64_MAX / nq) return B200_ERROR_INVALID_PARAM;
  for (const void* x : {q, k, v, (const void*)out})
    if (reinterpret_cast<uintptr_t>(x) & 15u) return B200_ERROR_INVALID_PARAM;
  if (reinterpret_cast<uintptr_t>(cu_seqlens) & 3u) return B200_ERROR_INVALID_PARAM;
  const int64_t qcols = (int64_t)(nq - 1) * q_head_stride + hd, kcols = (int64_t)(nkv - 1) * k_head_stride + hd,
                vcols = (int64_t)(nkv - 1) * v_head_stride + hdv;
  if (q_stride < qcols || k_stride < kcols || v_stride < vcols ||
      out_stride < (int64_t)(nq - 1) * out_head_stride + hdv)
    return B200_ERROR_INVALID_PARAM;
  if (num_seqs == 0 || max_seqlen == 0 || total_tokens == 0) return B200_OK;
  const bool pair_heads = nq / nkv % 2 == 0;
  const int rows = pair_heads ? kTile : 2 * kTile;
  // by tile where lengths are near each other: at most a quarter more numbers than by sequence, where they are level
  const int64_t by_tile = ((int64_t)max_seqlen + rows - 1) / rows * num_seqs, by_sequence = total_tokens / rows + num_seqs;
  const bool tiles = 4 * by_tile <= 5 * by_sequence;
  const int64_t items = (tiles ? by_tile : by_sequence) * (pair_heads ? nq / 2 : nq);
  if (total_tokens > INT32_MAX - 2 * kTile || qcols > INT32_MAX || kcols > INT32_MAX || vcols > INT32_MAX ||
      items > INT32_MAX - 4096 || max_seqlen > INT32_MAX - 2 * kTile)
    return B200_ERROR_UNSUPPORTED;
  // a window or sinks behind the longest prompt change nothing; kept small so that sums of positions fit
  window = std::min(window, max_seqlen);
  sinks = std::min(sinks, max_seqlen);
  const int grid = (int)std::min<int64_t>(items, sm_count());
  CUtensorMap mq, mk, mv;
  auto run = [&](auto prob, int cols) {
    prob.out = static_cast<__nv_bfloat16*>(out);
    prob.os = out_stride;
    prob.ohs = out_head_stride;
    prob.cu = cu_seqlens;
    prob.nq = nq;
    prob.nkv = nkv;
    prob.nseq = num_seqs;
    prob.items = (int)items;
    prob.max_rows = max_seqlen;
    prob.total = (int)total_tokens;
    prob.qhs = q_head_stride;
    prob.khs = k_head_stride;
    prob.vhs = v_head_stride;
    prob.scale_log2 = scale * 1.4426950408889634f;
    prob.window = window;
    prob.sinks = sinks;
    prob.out_cols = cols;
    prob.pair_heads = pair_heads;
    prob.by_tile = tiles;
    return launch_items(mq, mk, mv, prob, grid, stream);
  };
  if (hd < 64) {
    if (!make_map_heads(&mq, q, total_tokens, nq, hd, q_head_stride, q_stride) ||
        !make_map_heads(&mk, k, total_tokens, nkv, hd, k_head_stride, k_stride) ||
        !make_map_heads(&mv, v, total_tokens, nkv, hd, v_head_stride, v_stride))
      return B200_ERROR_UNSUPPORTED;
    return run(Window<64, 64, true>{}, hd);
  }
  if (!make_map(&mq, q, total_tokens, qcols, q_stride) || !make_map(&mk, k, total_tokens, kcols, k_stride) ||
      !make_map(&mv, v, total_tokens, vcols, v_stride))
    return B200_ERROR_UNSUPPORTED;
  if (hd == 192) return run(Window<192, 128, false>{}, hdv);
  if (hd == 128) return run(Window<128, 128, false>{}, hdv);
  return run(Window<64, 64, false>{}, hdv);
}

// Single-token attention over a paged KV cache with a sliding window and a few
// first tokens that stay visible (sinks), and, for the batch whose sequences
// share a prefix, the part of each sequence's own tokens, joined with the
// prefix's parts (PrefixParts in shared_prefix.h).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(q.k_j scale log2(e) - m),
//   over j < context with j >= context - window or j < sinks,
// in parts that each keep (m, sum, unnormalised output) and are joined by
//   m = max m_i, sum = sum_i 2^(m_i - m) sum_i, and the outputs alike.
//
// Every visible token's K and V are read once for up to 16 query heads that
// share them, 4 flops for each byte read and head: memory bounds it.  (Groups of
// more heads take a CTA for each 16, which mostly find the tiles in L2: 64
// sequences that show 4100 tokens of one 128-wide kv head take 34 us for 16 heads,
// 41 for 17 and for 32, 59 for 40 and for 64; the copy rate's floor is 20.)
// One CTA takes a stretch of the visible 64-token tiles of one (sequence, kv
// head); when there are too few pairs to fill the GPU, up to 8 CTAs of a
// cluster share a pair's tiles and join their parts through distributed shared
// memory, so there is no workspace, no second launch and nothing that two
// captured graphs could share.  Only tiles with a visible token are touched:
// table entries between the sinks and the window are never read, so their
// blocks may have been given to others.
//
// Inside a CTA a producer warp brings tiles in by TMA through a three-stage
// ring (32 KB a stage at 128-wide heads, two CTAs an SM); each of four warps
// takes 16 keys of a tile for up to 16 query heads (m16n8k16), with its own
// softmax state, joined at the end.  In a tile that is visible in part, value
// rows of hidden tokens are zeroed in shared memory before they are used, so a
// NaN or an infinity there (a block's unwritten rest, another sequence's data)
// does not reach the output.
//
// Measured: 64 sequences of up to 32768 tokens, window 4096, 32 / 8 heads of 128:
// 161 to 168 us for 1.055 GB, 96 % of the measured copy rate and more; heads of 64
// 82 us for half of that.  Two stages and three CTAs an SM took 229.  Contexts of
// a few tiles are bound by a CTA's way from its length to its table, tiles and
// join, 5 us: 64 of 512 tokens on average take 36 us for 129 MB.  (CTAs that walk
// many pairs, loading ahead, took 50: more registers, and joins in turns to fit
// two of them on an SM.)
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "shared_prefix.h"
#include "tensor_map.h"

using namespace b200;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;      // tokens per tile
constexpr int kBox = 64 * kTile * 2;  // a TMA box: 64 tokens x 64 dims
constexpr int kStages = 3;
constexpr int kRows = 16;      // query heads of a CTA (rows of the MMA)
constexpr int kThreads = 160;  // warps 0-3 compute, warp 4 loads
constexpr int kProducer = 4;
constexpr int kMaxCluster = 8;

template <int HD>
struct Cfg {
  static constexpr int BOXES = HD / 64;
  static constexpr int TILE = BOXES * kBox;
  static constexpr int STAGE = 2 * TILE;  // K, V
  static constexpr int Q_BYTES = kRows * HD * 2;
  static constexpr int BARS = kStages * STAGE + Q_BYTES;
  static constexpr int SMEM = BARS + 64 + 1024;
  // the parts are joined where the tiles were: four warps' outputs, their join, maxima and sums
  static_assert((kRows * HD * 5 + 10 * kRows) * 4 <= kStages * STAGE, "room for the join");
};

struct Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const int32_t* tables;
  int width;
  const int32_t* context;
  int nq, nkv, group, head_tiles, block_size;
  int64_t num_blocks;
  float scale_log2;
  int window, sinks;  // window >= width * block_size: all tokens
  __nv_bfloat16* out;
  int64_t out_stride;
  PrefixParts prefix;  // parts: nullptr without a shared prefix
  unsigned* err;
};

// Tiles with a visible token, in order: the sinks' and then the window's.
struct Tiles {
  int context, lo, sinks;  // visible: j < context and (j >= lo or j < sinks)
  int head, window_first, count;
  B200_DEV int at(int i) const { return i < head ? i : window_first + i - head; }
  B200_DEV bool whole(int tile) const {
    const int k = tile * kTile;
    return k + kTile <= context && (k >= lo || k + kTile <= sinks);
  }
  B200_DEV bool sees(int j) const { return j < context && (j >= lo || j < sinks); }
};

B200_DEV Tiles visible_tiles(int context, int window, int sinks) {
  Tiles t;
  t.context = context;
  t.lo = max(0, context - window);
  t.sinks = min(sinks, t.lo);
  t.window_first = t.lo / kTile;
  t.head = min((t.sinks + kTile - 1) / kTile, t.window_first);
  const int total = (context + kTile - 1) / kTile;
  t.count = t.head + max(0, total - t.window_first);
  return t;
}

// Byte offset of 16-byte chunk c of token row r in a tile of 64-dim boxes with the 128-byte swizzle.
B200_DEV uint32_t tile_off(int r, int c) {
  return (uint32_t)((c >> 3) * kBox + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// A float of CTA `rank`'s shared memory.
B200_DEV float cluster_load_f(uint32_t addr, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map(addr, (uint32_t)rank)) : "memory");
  return v;
}

B200_DEV float4 cluster_load_f4(uint32_t addr, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_map(addr, (uint32_t)rank))
               : "memory");
  return v;
}

template <int HD>
__global__ void __launch_bounds__(kThreads) paged_window_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                const __grid_constant__ CUtensorMap tmV,
                                                                const Params p) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + kStages * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);
  uint64_t* empty = full + kStages;

  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  int id = blockIdx.x / ctas;
  const int ht = id % p.head_tiles;
  id /= p.head_tiles;
  const int kh = id % p.nkv;
  const int b = id / p.nkv;
  const int head0 = kh * p.group + ht * kRows;  // first query head of this CTA
  const int rows = min(kRows, p.group - ht * kRows);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Behind the prefix kernel of the same call, only its parts have to be waited
  // for: it lets this kernel start after its own wait for all earlier ones.
  if (!p.prefix.parts) {
    pdl_trigger();
    pdl_wait();
  }
  int context = p.context[b];
  if (context < 0 || context > p.width * p.block_size) {
    if (threadIdx.x == 0) raise_error(p.err, DEV_ERR_BAD_INDEX);
    context = max(0, min(context, p.width * p.block_size));
  }
  const Tiles tiles = visible_tiles(context, p.window, p.sinks);
  const int share = (tiles.count + ctas - 1) / ctas;
  const int first = min(rank * share, tiles.count), n = min(share, tiles.count - first);

  // query rows, zeros up to 16
  for (int i = threadIdx.x; i < kRows * (HD / 8); i += kThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) v = *reinterpret_cast<const uint4*>(p.q + (int64_t)b * p.q_stride + (int64_t)(head0 + r) * HD + c * 8);
    *reinterpret_cast<uint4*>(sQ + r * HD * 2 + ((c ^ (r & 7)) << 4)) = v;
  }
  __syncthreads();

  float o[HD / 8][4];
#pragma unroll
  for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  if (warp == kProducer) {
    // lane l looks up the block of tile 32 k + l; lane 0 issues the copies
    int my_row = 0, i = 0;
    bool ok = true;
    for (; i < n; ++i) {
      const int s = i % kStages, round = i / kStages;
      if (lane == 0 && round > 0) ok = mbar_wait(&empty[s], (round - 1) & 1, p.err);
      if (!(ok = __shfl_sync(0xffffffffu, ok, 0))) break;
      if ((i & 31) == 0 && i + lane < n) {
        const int tok = tiles.at(first + i + lane) * kTile;
        int blk = p.tables[(int64_t)b * p.width + tok / p.block_size];
        if (blk < 0 || blk >= p.num_blocks) {
          raise_error(p.err, DEV_ERR_BAD_INDEX);
          blk = 0;
        }
        my_row = (blk * p.nkv + kh) * p.block_size + tok % p.block_size;
      }
      const int row = __shfl_sync(0xffffffffu, my_row, i & 31);
      if (lane == 0) {
        uint8_t* dst = smem + s * C::STAGE;
        mbar_arrive_expect_tx(&full[s], C::STAGE);
#pragma unroll
        for (int x = 0; x < C::BOXES; ++x) {
          tma_load_2d(dst + x * kBox, &tmK, &full[s], 64 * x, row);
          tma_load_2d(dst + C::TILE + x * kBox, &tmV, &full[s], 64 * x, row);
        }
      }
      __syncwarp();
    }
    // whoever gives up before using a tile: every copy has landed before its memory is used again
    if (lane == 0)
      for (int k = max(0, i - kStages); k < i; ++k) mbar_wait(&full[k % kStages], (k / kStages) & 1, p.err);
    __syncwarp();
  } else {
    uint32_t qf[HD / 16][4];
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      const int mat = lane >> 3;
      const int r = (lane & 7) + ((mat & 1) ? 8 : 0);
      const int c = kk * 2 + (mat >> 1);
      ldmatrix_x4(qf[kk], smem_u32(sQ + r * HD * 2 + ((c ^ (r & 7)) << 4)));
    }
    for (int i = 0; i < n; ++i) {
      const int s = i % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (i / kStages) & 1, p.err))) break;  // a warp as a whole
      uint8_t* sK = smem + s * C::STAGE;
      uint8_t* sV = sK + C::TILE;
      float sc[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const int mat = lane >> 3;
        const int r = warp * 16 + (mat >> 1) * 8 + (lane & 7);
        const int c = kk * 2 + (mat & 1);
        uint32_t bf[4];
        ldmatrix_x4(bf, smem_u32(sK + tile_off(r, c)));
        mma_bf16_16816(sc[0], qf[kk], bf);
        mma_bf16_16816(sc[1], qf[kk], bf + 2);
      }
      const int tile = tiles.at(first + i);
      const int k0 = tile * kTile + warp * 16;  // this warp's first key
      const bool part = !tiles.whole(tile);
      if (part) {
        // hidden tokens' value rows, two lanes a row
        const int r = warp * 16 + (lane >> 1);
        if (!tiles.sees(k0 + (lane >> 1)))
#pragma unroll
          for (int c = 0; c < HD / 16; ++c)
            *reinterpret_cast<uint4*>(sV + tile_off(r, (lane & 1) * (HD / 16) + c)) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = sc[j][e] * p.scale_log2;
          if (part && !tiles.sees(k0 + j * 8 + 2 * t4 + (e & 1))) x = -INFINITY;
          sc[j][e] = x;
          mx[e >> 1] = fmaxf(mx[e >> 1], x);
        }
      float corr[2], base[2], rs[2] = {0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float m_new = fmaxf(m_run[r], mx[r]);
        corr[r] = m_new == -INFINITY ? 1.f : exp2f(m_run[r] - m_new);
        base[r] = m_new == -INFINITY ? 0.f : m_new;
        m_run[r] = m_new;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[j][e] = exp2f(sc[j][e] - base[e >> 1]);
          rs[e >> 1] += sc[j][e];
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) l_run[r] = l_run[r] * corr[r] + rs[r];
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) {
        o[j][0] *= corr[0];
        o[j][1] *= corr[0];
        o[j][2] *= corr[1];
        o[j][3] *= corr[1];
      }
      // P in 16 bits: the rounding (2^-9 of a weight at most) is that of the products' operand type
      const uint32_t pa[4] = {pack2(sc[0][0], sc[0][1]), pack2(sc[0][2], sc[0][3]), pack2(sc[1][0], sc[1][1]),
                              pack2(sc[1][2], sc[1][3])};
#pragma unroll
      for (int jp = 0; jp < HD / 16; ++jp) {
        const int mat = lane >> 3;
        const int r = warp * 16 + (mat & 1) * 8 + (lane & 7);
        const int c = 2 * jp + (mat >> 1);
        uint32_t bf[4];
        ldmatrix_x4_trans(bf, smem_u32(sV + tile_off(r, c)));
        mma_bf16_16816(o[2 * jp], pa, bf);
        mma_bf16_16816(o[2 * jp + 1], pa, bf + 2);
      }
      if (part) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros, before a copy lands there
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
  }

  // ---- this CTA's part: the four warps joined, in shared memory ----
  __syncthreads();  // every copy has landed, and been used where no wait ran out
  float* sm = reinterpret_cast<float*>(smem);  // [4][16] maxima
  float* sl = sm + 64;                         // [4][16] sums
  float* part_m = sl + 64;                     // [16] joined maxima
  float* part_l = part_m + 16;                 // [16] joined sums
  float* part_o = part_l + 16;                 // [16][HD] joined outputs
  float* warp_o = part_o + kRows * HD;         // [4][16][HD]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
  }
  if (warp < 4) {
    if (t4 == 0) {
      sm[warp * 16 + g] = m_run[0];
      sm[warp * 16 + g + 8] = m_run[1];
      sl[warp * 16 + g] = l_run[0];
      sl[warp * 16 + g + 8] = l_run[1];
    }
    float* wo = warp_o + warp * kRows * HD;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      *reinterpret_cast<float2*>(wo + g * HD + j * 8 + 2 * t4) = make_float2(o[j][0], o[j][1]);
      *reinterpret_cast<float2*>(wo + (g + 8) * HD + j * 8 + 2 * t4) = make_float2(o[j][2], o[j][3]);
    }
  }
  __syncthreads();
  const bool alone = ctas == 1 && !p.prefix.parts;
  for (int i = threadIdx.x; i < rows * HD; i += kThreads) {
    const int row = i / HD;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w * 16 + row]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(sm[w * 16 + row] - ref);  // 0 for a warp without a visible key
      L += f * sl[w * 16 + row];
      acc += f * warp_o[(w * kRows + row) * HD + i % HD];
    }
    if (alone) {  // this CTA's part is all there is
      // an empty context gives zeros; where it is not empty, scores of -inf alone are 0 / 0
      p.out[(int64_t)b * p.out_stride + (int64_t)head0 * HD + i] = f2bf(context == 0 ? 0.f : acc / L);
      continue;
    }
    part_o[i] = acc;
    if (i % HD == 0) {
      part_m[row] = M;
      part_l[row] = L;
    }
  }
  if (alone) return;
  if (ctas > 1) cluster_sync();
  else __syncthreads();

  // ---- the parts of the cluster, and the prefix's, joined ----
  // The weights of a row's parts, 2^(m_i - M) over the weighted sum, a row a warp;
  // then a share of the outputs each, four at a time.  (A prefix's parts are
  // divided by their sums already: the weight of their log sum is all they need.)
  if (p.prefix.parts) pdl_wait();
  const PrefixSpan span = p.prefix.parts ? prefix_span(p.prefix, b, kh, p.nkv, ht * kRows, HD) : PrefixSpan{};
  const uint32_t am = smem_u32(part_m), al = smem_u32(part_l), ao = smem_u32(part_o);
  const int parts = ctas + span.count;
  float* weight = warp_o;  // [rows][parts]: the warps' outputs are joined
  for (int row = warp; row < rows; row += kThreads / 32) {
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32)
      M = fmaxf(M, i < ctas ? cluster_load_f(am + 4 * row, i) : span.lse[(i - ctas) * 256 + row]);
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int i = lane; i < parts; i += 32) {
      const float f = exp2f((i < ctas ? cluster_load_f(am + 4 * row, i) : span.lse[(i - ctas) * 256 + row]) - ref);
      weight[row * parts + i] = f;
      L += i < ctas ? f * cluster_load_f(al + 4 * row, i) : f;
    }
    L = warp_sum(L);
    // nothing visible: zeros; scores of -inf alone: 0 / 0
    const float inv = L > 0.f ? 1.f / L : context == 0 && span.count == 0 ? 0.f : NAN;
    for (int i = lane; i < parts; i += 32) weight[row * parts + i] *= inv;
  }
  __syncthreads();
  for (int v = rank * kThreads + threadIdx.x; v < rows * HD / 4; v += ctas * kThreads) {
    const int row = v / (HD / 4);
    const float* w = weight + row * parts;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float f, const float4& o) {
      acc.x = fmaf(f, o.x, acc.x);
      acc.y = fmaf(f, o.y, acc.y);
      acc.z = fmaf(f, o.z, acc.z);
      acc.w = fmaf(f, o.w, acc.w);
    };
    for (int r = 0; r < ctas; ++r) add(w[r], cluster_load_f4(ao + 16 * v, r));
    const float4* po = reinterpret_cast<const float4*>(span.parts) + v;
#pragma unroll 8
    for (int k = 0; k < span.count; ++k) add(w[ctas + k], __ldcg(po + (int64_t)k * 64 * HD));
    __nv_bfloat16* o = p.out + (int64_t)b * p.out_stride + (int64_t)head0 * HD + 4 * v;
    const uint2 packed = make_uint2(pack2(acc.x, acc.y), pack2(acc.z, acc.w));
    if ((reinterpret_cast<uintptr_t>(o) & 7u) == 0) {
      *reinterpret_cast<uint2*>(o) = packed;
    } else {
      const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&packed);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = e[i];
    }
  }
  if (p.prefix.parts) pdl_trigger();
  if (ctas > 1) cluster_sync();  // the parts stay until they are read
}

// The cache viewed as a [rows, HD] bf16 matrix, box = 64 rows x 64 dims.
template <int HD>
bool make_cache_map(CUtensorMap* m, const void* ptr, int64_t rows) {
  return encode_tiled_2d(m, ptr, HD, rows, HD * 2, 64, kTile);
}

// CTAs that share a (sequence, kv head, head tile): none but one when these
// fill the GPU with two CTAs an SM by themselves, else so many that they do, at
// most 8 and never more than the tiles that a sequence can show.  Eight kv heads
// of 128, 1028 tokens shown, with 1, 2, 4 and 8 CTAs a pair: one sequence 16.6,
// 12.7, 10.4 and 9.5 us; eight (two CTAs an SM with 4) 18.1, 15.8, 14.3 and 23.2;
// sixteen (with 2) 21.5, 19.6, 28.0 and 44.2.  At 8196 tokens one takes 84, 46, 27
// and 18.5; at 300 tokens the number hardly matters (6.7 to 7.2).
unsigned cluster_for(int64_t pairs, int max_tiles) {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (sms <= 0) sms = 148;
  unsigned c = 1;
  while (c < kMaxCluster && pairs * c * 2 <= 2 * sms && (int)(2 * c) <= max_tiles) c *= 2;
  return c;
}

template <int HD>
int launch(const Params& p, const void* k_cache, const void* v_cache, int64_t rows, unsigned ctas, int64_t pairs,
           cudaStream_t stream) {
  auto k = paged_window_kernel<HD>;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERROR_UNSUPPORTED;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    done[dev] = true;
  }
  CUtensorMap tk, tv;
  if (!make_cache_map<HD>(&tk, k_cache, rows) || !make_cache_map<HD>(&tv, v_cache, rows)) return B200_ERROR_UNSUPPORTED;
  launch_clusters(k, ctas, dim3((unsigned)(pairs * ctas)), kThreads, Cfg<HD>::SMEM, stream, tk, tv, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool al4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

namespace b200 {

int paged_window_check(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                       const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
                       int nq, int nkv, int head_dim, int block_size, int64_t num_blocks, float scale, const void* out,
                       int64_t out_stride, int max_context) {
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out || batch < 0 || nq <= 0 || nkv <= 0 ||
      nq % nkv || max_blocks_per_seq <= 0 || num_blocks <= 0 || max_context < 0 ||
      !(scale > 0.f && scale < INFINITY))
    return B200_ERROR_INVALID_PARAM;
  if ((head_dim != 64 && head_dim != 128) || (block_size != 64 && block_size != 128)) return B200_ERROR_UNSUPPORTED;
  if (q_stride % 8 || q_stride < (int64_t)nq * head_dim || out_stride < (int64_t)nq * head_dim || !al16(q) ||
      !al16(k_cache) || !al16(v_cache) || !al4(block_tables) || !al4(context_lens) ||
      (reinterpret_cast<uintptr_t>(out) & 1u))
    return B200_ERROR_INVALID_PARAM;
  if ((int64_t)max_blocks_per_seq * block_size < max_context) return B200_ERROR_INVALID_PARAM;
  if ((int64_t)max_blocks_per_seq * block_size > INT32_MAX - 256 || num_blocks > INT32_MAX / block_size / nkv ||
      (int64_t)batch * nq > INT32_MAX / kMaxCluster)
    return B200_ERROR_UNSUPPORTED;
  return B200_OK;
}

int paged_window_launch(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                        const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
                        int nq, int nkv, int head_dim, int block_size, int64_t num_blocks, float scale, int window,
                        int sinks, void* out, int64_t out_stride, int max_context, const PrefixParts& prefix,
                        cudaStream_t stream) {
  const int room = max_blocks_per_seq * block_size;
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.tables = block_tables;
  p.width = max_blocks_per_seq;
  p.context = context_lens;
  p.nq = nq;
  p.nkv = nkv;
  p.group = nq / nkv;
  p.head_tiles = (p.group + kRows - 1) / kRows;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.scale_log2 = scale * kLog2e;
  p.window = std::min(window, room);
  p.sinks = std::min(sinks, room);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.prefix = prefix;
  int dev = 0;
  cudaGetDevice(&dev);
  p.err = error_word(dev);
  // tiles that the longest sequence shows: the window may cut through two tiles at its ends
  const int64_t seen = std::min<int64_t>(max_context, (int64_t)p.window + p.sinks);
  const int max_tiles = (int)std::min<int64_t>((max_context + kTile - 1) / kTile, seen / kTile + 2);
  const int64_t pairs = (int64_t)batch * nkv * p.head_tiles;
  const unsigned ctas = cluster_for(pairs, max_tiles);
  const int64_t rows = num_blocks * nkv * block_size;
  return head_dim == 128 ? launch<128>(p, k_cache, v_cache, rows, ctas, pairs, stream)
                         : launch<64>(p, k_cache, v_cache, rows, ctas, pairs, stream);
}

}  // namespace b200

extern "C" int b200_paged_decode_window(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                                        const int32_t* block_tables, int max_blocks_per_seq,
                                        const int32_t* context_lens, int batch, int nq, int nkv, int head_dim,
                                        int block_size, int64_t num_blocks, float scale, int window, int sinks,
                                        void* out, int64_t out_stride, int max_context, b200_stream_t stream) {
  if (window <= 0 || sinks < 0) return B200_ERROR_INVALID_PARAM;
  const int rc = b200::paged_window_check(q, q_stride, k_cache, v_cache, block_tables, max_blocks_per_seq,
                                          context_lens, batch, nq, nkv, head_dim, block_size, num_blocks, scale, out,
                                          out_stride, max_context);
  if (rc != B200_OK || batch == 0) return rc;
  return b200::paged_window_launch(q, q_stride, k_cache, v_cache, block_tables, max_blocks_per_seq, context_lens,
                                   batch, nq, nkv, head_dim, block_size, num_blocks, scale, window, sinks, out,
                                   out_stride, max_context, b200::PrefixParts{}, stream);
}

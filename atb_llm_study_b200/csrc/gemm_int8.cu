// 8-bit integer GEMM on the 5th-generation tensor cores:
//   C[m, n] = epi(a_scale[m] * b_scale[n] * sum_k A[m, k] B[n, k])
// with int8 operands, exact 32-bit integer sums and one rounding to bf16.
//
// Three kernels, each with a TMA producer warp, an MMA issuer thread and
// epilogue warps around a ring of shared-memory stages (128-byte swizzle):
//   gemm_i8_pair_kernel   many tokens: persistent CTA pairs, 256 x 256 tiles
//                         (cta_group::2), two TMEM accumulators; also grouped.
//   gemm_i8_split_kernel  few tokens: weights on the 128-row MMA side, tokens on
//                         the N side, K split over a cluster.
//   gemm_i8_group_kernel  few tokens per expert: weights on the 128-row side,
//                         one persistent CTA per SM over all experts' tiles.
//
// Nothing is loaded before the previous kernel on the stream has finished: the
// weights can be that kernel's output (the row quantisation makes them).
// TMEM is allocated after that wait and the next kernel released after the
// allocation: two kernels of which one holds TMEM the other needs never wait
// for one another.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"

using namespace b200;

namespace {

constexpr int BM = 128;
constexpr int BK = 128;  // bytes of K per stage: the swizzle span
constexpr int kThreads = 192;
constexpr int kMaxGroups = 256;                           // experts of one grouped GEMM
constexpr int kGroupTabBytes = 2 * (kMaxGroups + 2) * 4;  // row offsets + unit prefix in shared memory
// The largest |sum| is 128 * 128 * K (both operands may hold -128): it fits 31 bits up to here.
constexpr int64_t kMaxK = 131056;

struct Params {
  int64_t rows;  // MMA M extent
  int64_t cols;  // MMA N extent
  int tiles_m, tiles_n, kb_total, kb_per_split;
  const float* row_scale;  // of the MMA rows / columns (tokens or features by orientation)
  const float* col_scale;
  __nv_bfloat16* C;
  int64_t ldc;
  const __nv_bfloat16* bias;
  const __nv_bfloat16* R;
  int64_t ldr;
  unsigned* err;
  // Grouped: the tokens of group g are rows [goff[g], goff[g+1]) and its
  // weights rows [g*gN, (g+1)*gN).
  const int32_t* goff;
  int groups;
  int64_t gN;
  int gF;
  int64_t gRows;
};

struct Unit {
  int tok0, wrow0;  // TMA rows of the token and the weight operand
  int feat0;        // first output column
  int tok_lim, feat_lim;
  int n;            // grouped pairs: tokens of this tile, rounded up to a multiple of 32
};

// 0.5 x (1 + tanh(u)) = x / (1 + e^-2u), u = sqrt(2/pi) (x + 0.044715 x^3): one
// exponential and one division where tanhf costs several times that, and no
// cancellation for negative x.
__device__ __forceinline__ float gelu_tanh_f(float x) {
  return __fdividef(x, 1.f + __expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
}
__device__ __forceinline__ float silu_f(float x) { return __fdividef(x, 1.f + __expf(-x)); }

constexpr bool has_bias(int e) {
  return e == B200_EPI_BIAS || e == B200_EPI_BIAS_GELU || e == B200_EPI_BIAS_RESIDUAL;
}
constexpr bool has_residual(int e) { return e == B200_EPI_RESIDUAL || e == B200_EPI_BIAS_RESIDUAL; }

__device__ __forceinline__ void add4(float v[4], const __nv_bfloat16* src) {
  const uint2 u = *reinterpret_cast<const uint2*>(src);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  v[0] += a.x, v[1] += a.y, v[2] += b.x, v[3] += b.y;
}

// Unit w of a grouped launch over tiles of TOKT tokens x FEATT features.
// gtab[0..G] holds the groups' token row offsets and gtab[G+1..2G+1] the prefix
// of their unit counts; within a group the token tiles of one feature tile are
// consecutive (they share that weight tile).
template <int TOKT, int FEATT>
__device__ __forceinline__ Unit group_unit(int w, const Params& p, const int* gtab) {
  const int* up = gtab + p.groups + 1;
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (up[mid] <= w) lo = mid;
    else hi = mid;
  }
  const int t0 = gtab[lo], t1 = gtab[lo + 1];
  const int r = w - up[lo];
  const int tt = (t1 - t0 + TOKT - 1) / TOKT;
  Unit u;
  u.tok0 = t0 + r % tt * TOKT;
  u.feat0 = r / tt * FEATT;
  u.wrow0 = (int)(lo * p.gN) + u.feat0;
  u.tok_lim = t1;
  u.feat_lim = (int)p.gN;
  u.n = min(TOKT, (t1 - u.tok0 + 31) & ~31);
  return u;
}

// A producer that gives up waits (again with a limit) for its copies in flight:
// the last `stages` of the `issued` ones.
__device__ __forceinline__ void drain_loads(uint64_t* full, int stages, int issued, unsigned* err) {
  for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, err);
}

// One warp fills gtab from the device offsets, 32 groups at a time (prefix
// maximum and prefix sum); offsets that fall or leave [0, rows] are clamped and
// reported.
template <int TOKT>
__device__ __forceinline__ void fill_group_table(int* gtab, const Params& p, int lane) {
  constexpr int kRounds = (kMaxGroups + 1 + 31) / 32;
  int v[kRounds];  // all loads at once
#pragma unroll
  for (int i = 0; i < kRounds; ++i) v[i] = i * 32 + lane <= p.groups ? p.goff[i * 32 + lane] : 0;
  int prev = 0, run = 0;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (i * 32 > p.groups) break;
    const int g = i * 32 + lane;
    int x = g == 0 ? 0 : max(v[i], prev);
    int before = __shfl_up_sync(0xffffffffu, v[i], 1);
    if (lane == 0) before = i == 0 ? 0 : prev;
    if (g <= p.groups && (v[i] < before || v[i] > p.gRows || v[i] < 0 || (g == 0 && v[i] != 0)))
      raise_error(p.err, DEV_ERR_BAD_INDEX);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = max(x, y);
    }
    x = min(x, (int)p.gRows);
    int lo = __shfl_up_sync(0xffffffffu, x, 1);
    if (lane == 0) lo = prev;
    int sum = g > 0 && g <= p.groups ? (x - lo + TOKT - 1) / TOKT * p.gF : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    sum += run;
    if (g <= p.groups) {
      gtab[g] = x;
      gtab[p.groups + 1 + g] = sum;
    }
    prev = __shfl_sync(0xffffffffu, x, 31);
    run = __shfl_sync(0xffffffffu, sum, 31);
  }
}

// CW (16 or 32) accumulator columns, tokens tok0.., of 32 consecutive feature
// rows (one a lane, the first at output feature feat0 of the untiled width),
// through the epilogue and transposed among the lanes, so that a lane stores
// four features of a token at once and a warp's store covers whole 32-byte
// sectors.  ts: the tokens' scales; fscale: this lane's feature's.
template <int EPI, int CW>
__device__ __forceinline__ void emit_features(const uint32_t acc[CW], int feat0, int tok0, float fscale, const float* ts,
                                              const Unit& u, int lane, const Params& p) {
  float v[CW];
#pragma unroll
  for (int i = 0; i < CW; i += 4) {
    const float4 s = *reinterpret_cast<const float4*>(ts + i);
    v[i] = (float)(int)acc[i] * fscale * s.x;
    v[i + 1] = (float)(int)acc[i + 1] * fscale * s.y;
    v[i + 2] = (float)(int)acc[i + 2] * fscale * s.z;
    v[i + 3] = (float)(int)acc[i + 3] * fscale * s.w;
  }
  constexpr unsigned kAll = 0xffffffffu;
  const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
  if (EPI == B200_EPI_SWIGLU) {
    // lanes 2j / 2j+1 hold gate / up of output j: the even lane finishes the
    // first half of the tokens, the odd lane the second
    constexpr int H = CW / 2;
    float o[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float other = __shfl_xor_sync(kAll, b0 ? v[i] : v[H + i], 1);
      o[i] = b0 ? silu_f(other) * v[H + i] : silu_f(v[i]) * other;
    }
    uint32_t a[H / 2];  // two outputs of token 2t + b1
#pragma unroll
    for (int t = 0; t < H / 2; ++t) {
      const float got = __shfl_xor_sync(kAll, b1 ? o[2 * t] : o[2 * t + 1], 2);
      a[t] = b1 ? pack2(got, o[2 * t + 1]) : pack2(o[2 * t], got);
    }
    const int f = feat0 / 2 + (lane >> 1 & ~3);
#pragma unroll
    for (int t = 0; t < H / 4; ++t) {  // four outputs of token 4t + 2 b2 + b1
      const uint32_t got = __shfl_xor_sync(kAll, b2 ? a[2 * t] : a[2 * t + 1], 4);
      const uint2 w = b2 ? make_uint2(got, a[2 * t + 1]) : make_uint2(a[2 * t], got);
      const int64_t tok = tok0 + (b0 ? H : 0) + 4 * t + 2 * b2 + b1;
      if (2 * f < u.feat_lim && tok < u.tok_lim) *reinterpret_cast<uint2*>(p.C + tok * p.ldc + f) = w;
    }
    return;
  }
  uint32_t a[CW / 2];  // two features of token 2t + b0
#pragma unroll
  for (int t = 0; t < CW / 2; ++t) {
    const float got = __shfl_xor_sync(kAll, b0 ? v[2 * t] : v[2 * t + 1], 1);
    a[t] = b0 ? pack2(got, v[2 * t + 1]) : pack2(v[2 * t], got);
  }
  const int f = feat0 + (lane & ~3);
#pragma unroll
  for (int t = 0; t < CW / 4; ++t) {  // four features of token 4t + 2 b1 + b0
    const uint32_t got = __shfl_xor_sync(kAll, b1 ? a[2 * t] : a[2 * t + 1], 2);
    const uint2 w = b1 ? make_uint2(got, a[2 * t + 1]) : make_uint2(a[2 * t], got);
    const int64_t tok = tok0 + 4 * t + 2 * b1 + b0;
    if (f < u.feat_lim && tok < u.tok_lim) *reinterpret_cast<uint2*>(p.C + tok * p.ldc + f) = w;
  }
}

// ---------------------------------------------------------------------------
// Many tokens: persistent CTA pairs.  CTA r of a pair loads 128 token rows and
// 128 weight rows of each k-block; the leader (rank 0) issues M = 256, N = 256
// MMAs that read both halves, and each CTA's epilogue drains its 128 token rows
// from its own TMEM.  Against single CTAs with 128 x 256 tiles a pair moves a
// third less through L2 and shared memory per product.
//
// 16384 x 4096 x 12288 with residual: 496 us alone, 3.3 POP/s; the tensor pipe is
// active in 90 % of the cycles that the SMs are (ncu), and a k-block takes 559
// cycles against the MMAs' 512.  What is left of those cycles is shared memory
// (32 KB in and as much out of it per 512 cycles) and the epilogue's use of it:
// 611 cycles with SwiGLU at K = 4096, 560 with an epilogue that does nothing.  Run
// back to back the power limit decides: 540 to 600 us at 1.5 GHz.
//
// Grouped launches come in two forms.  kRows is the plain one with a group's
// rows past its end not stored.  kCols turns the operands round: 256 weight rows
// on the M side and the group's tokens on the N side, whose extent can be any
// multiple of 32, so that small groups do no products for rows they lack.
// ---------------------------------------------------------------------------
constexpr int kPairTile = 256;
constexpr int kPairGroup = 8;  // token tiles walked per feature tile
constexpr int kPairStages = 6;
constexpr int kPairEpiWarps = 8;
constexpr int kParts = kPairEpiWarps / 4;         // warps over the columns (the four TMEM lane quarters over the rows)
constexpr int kPartCols = kPairTile / kParts;
constexpr int kPartChunks = kPartCols / 32;
constexpr int kPairThreads = 64 + kPairEpiWarps * 32;
constexpr int kPairStageBytes = 2 * BM * BK;  // of each CTA
constexpr int kPairColBytes = kPairEpiWarps * kPartCols * 2 * 4;  // column scales and biases of each epilogue warp
constexpr int kPairSmem = kPairStages * kPairStageBytes + 1024 /*align*/ + 256 /*barriers*/ + kPairColBytes + kGroupTabBytes;
constexpr int kTokBox = 64;  // token rows of one TMA box of a grouped launch

// 32 accumulator columns of one token row through the epilogue; scale and bias
// of the columns come from shared memory.  A lane has a row of its own, so each
// of a warp's stores (and residual loads) touches 32 lines and costs the L1 that
// the MMA operands pass through as many cycles, whatever its width: with `wide`
// (32-byte aligned rows) it moves 32 bytes at a time, otherwise 16 or 8.
template <int EPI>
__device__ __forceinline__ void emit_row(const uint32_t acc[32], int64_t tok, int feat0, float rscale, const float* cscale,
                                         const float* cbias, bool wide, const Unit& u, const Params& p) {
  constexpr bool kSwiglu = EPI == B200_EPI_SWIGLU;
  constexpr int W = kSwiglu ? 32 : 16;  // columns behind 32 bytes of output
#pragma unroll
  for (int g = 0; g < 32; g += W) {
    const int c0 = feat0 + g;
    if (c0 >= u.feat_lim) continue;
    const bool whole = wide && c0 + W <= u.feat_lim;
    const __nv_bfloat16* res = has_residual(EPI) ? p.R + tok * p.ldr + c0 : nullptr;
    Words8 r8;
    if (has_residual(EPI)) {
      if (whole) {
        r8 = load_32(res);
      } else {
        const uint4 lo = *reinterpret_cast<const uint4*>(res);
        const uint4 hi = c0 + 8 < u.feat_lim ? *reinterpret_cast<const uint4*>(res + 8) : make_uint4(0, 0, 0, 0);
        r8.w[0] = lo.x, r8.w[1] = lo.y, r8.w[2] = lo.z, r8.w[3] = lo.w;
        r8.w[4] = hi.x, r8.w[5] = hi.y, r8.w[6] = hi.z, r8.w[7] = hi.w;
      }
    }
    Words8 o;
#pragma unroll
    for (int h = 0; h < W; h += 4) {
      const float4 s = *reinterpret_cast<const float4*>(cscale + g + h);
      float x[4] = {(float)(int)acc[g + h] * rscale * s.x, (float)(int)acc[g + h + 1] * rscale * s.y,
                    (float)(int)acc[g + h + 2] * rscale * s.z, (float)(int)acc[g + h + 3] * rscale * s.w};
      if (has_bias(EPI)) {
        const float4 b = *reinterpret_cast<const float4*>(cbias + g + h);
        x[0] += b.x, x[1] += b.y, x[2] += b.z, x[3] += b.w;
      }
      if (EPI == B200_EPI_BIAS_GELU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = gelu_tanh_f(x[i]);
      }
      if (kSwiglu) {
        o.w[h / 4] = pack2(silu_f(x[0]) * x[1], silu_f(x[2]) * x[3]);
        continue;
      }
      if (has_residual(EPI)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r8.w[h / 2 + i]));
          x[2 * i] += r.x, x[2 * i + 1] += r.y;
        }
      }
      o.w[h / 2] = pack2(x[0], x[1]);
      o.w[h / 2 + 1] = pack2(x[2], x[3]);
    }
    __nv_bfloat16* out = p.C + tok * p.ldc + (kSwiglu ? c0 / 2 : c0);
    if (whole) {
      store_32(out, o);
    } else if (kSwiglu) {  // a pair of 8-byte halves for each 16 columns
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c0 + 8 * i < u.feat_lim) *reinterpret_cast<uint2*>(out + 4 * i) = make_uint2(o.w[2 * i], o.w[2 * i + 1]);
    } else {
      *reinterpret_cast<uint4*>(out) = make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
      if (c0 + 8 < u.feat_lim) *reinterpret_cast<uint4*>(out + 8) = make_uint4(o.w[4], o.w[5], o.w[6], o.w[7]);
    }
  }
}

// MODE: kPlain, kRows (grouped, tokens on the M side) or kCols (grouped, tokens on the N side).
constexpr int kPlain = 0, kRows = 1, kCols = 2;
template <int EPI, int MODE>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const Params p) {
  constexpr bool GROUPED = MODE != kPlain, COLS = MODE == kCols;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kPairStages * BM * BK;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairStages * kPairStageBytes);  // the leader's are used
  uint64_t* empty = full + kPairStages;
  uint64_t* tfull = empty + kPairStages;
  uint64_t* tempty = tfull + 2;  // the leader's are used
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* cols = reinterpret_cast<float*>(smem + kPairStages * kPairStageBytes + 256);
  int* gtab = reinterpret_cast<int*>(smem + kPairStages * kPairStageBytes + 256 + kPairColBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  int units = p.tiles_m * p.tiles_n;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kPairEpiWarps);
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  pdl_wait();
  if (GROUPED && warp == 0) fill_group_table<kPairTile>(gtab, p, lane);
  if (warp == 1) tmem_alloc_pair(tmem_slot, 2 * kPairTile);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers are ready, and both have their TMEM
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  if (GROUPED) units = gtab[2 * p.groups + 1];

  auto unit_at = [&](int w) {
    if (GROUPED) return group_unit<kPairTile, kPairTile>(w, p, gtab);
    const int span = kPairGroup * p.tiles_n;
    const int first = w / span * kPairGroup;
    const int gm = min(p.tiles_m - first, kPairGroup);
    const int r = w % span;
    Unit u;
    u.tok0 = (first + r % gm) * kPairTile;
    u.feat0 = u.wrow0 = r / gm * kPairTile;
    u.tok_lim = (int)p.rows;
    u.feat_lim = (int)p.cols;
    return u;
  };

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int w = pair; w < units && !*abort_flag; w += pairs) {
        const Unit u = unit_at(w);
        // rows of this CTA's half of both operands
        const int a_row = (COLS ? u.wrow0 : u.tok0) + rank * BM;
        const int b_row = COLS ? u.tok0 + rank * (u.n / 2) : u.wrow0 + rank * BM;
        const int boxes = COLS ? (u.n / 2 + kTokBox - 1) / kTokBox : 1;
        constexpr int box_bytes = (COLS ? kTokBox : BM) * BK;
        for (int kb = 0; kb < p.kb_total; ++kb, ++issued) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.err)) {
            *abort_flag = 1;
            break;
          }
          // the leader expects both CTAs' bytes; the other's may land first
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * (BM * BK + boxes * box_bytes));
          const uint32_t bar = cluster_map(smem_u32(&full[stage]), 0);
          tma_load_2d_pair(sA + stage * BM * BK, &tmA, bar, kb * BK, a_row);
          for (int i = 0; i < boxes; ++i)
            tma_load_2d_pair(sB + stage * BM * BK + i * box_bytes, &tmB, bar, kb * BK, b_row + i * kTokBox);
          if (++stage == kPairStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // the leader's barriers count both CTAs' copies; the other CTA leaves after it
      if (*abort_flag && rank == 0) drain_loads(full, kPairStages, issued, p.err);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader) ----------------
    if (lane == 0 && rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      int next_n = COLS && pair < units ? unit_at(pair).n : kPairTile;
      for (int w = pair; w < units && !*abort_flag; w += pairs, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, p.err)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t idesc = idesc_i8_s32(256, next_n);
        bool ok = true;
        for (int kb = 0; kb < p.kb_total; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * BM * BK);
          const uint32_t b0 = smem_u32(sB + stage * BM * BK);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_i8_pair(tmem_base + acc * kPairTile, smem_desc_k128(a0 + k * 32), smem_desc_k128(b0 + k * 32),
                         idesc, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&empty[stage]);
          // the next tile's extent is looked up while this one's products run
          if (COLS && kb == 0 && w + pairs < units) next_n = unit_at(w + pairs).n;
          if (++stage == kPairStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        umma_commit_pair(&tfull[acc]);
        if (!ok) {
          *abort_flag = 1;
          break;
        }
      }
      if (*abort_flag) {  // products in flight end before the operands' memory and TMEM go
        umma_commit_pair(drained);
        mbar_wait(drained, 0, p.err);
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const int part = (warp - 2) >> 2;
    float* cscale = cols + (warp - 2) * 2 * kPartCols;
    float* cbias = cscale + kPartCols;
    const bool wide = ((reinterpret_cast<uintptr_t>(p.C) | reinterpret_cast<uintptr_t>(p.R)) & 31) == 0 &&
                      p.ldc % 16 == 0 && (!has_residual(EPI) || p.ldr % 16 == 0);
    // what a unit's epilogue reads besides its sums is loaded a unit ahead
    struct Ahead {
      Unit u;
      float lane_scale;                              // this lane's row: token (feature with COLS)
      float scale[kPartChunks], bias[kPartChunks];   // column 32 i + lane of the warp's
    };
    const auto ahead = [&](int w) {
      Ahead n;
      n.u = unit_at(w);
      n.lane_scale = 0.f;
      const int r = rank * BM + q * 32 + lane;
      if (COLS ? n.u.feat0 + r < n.u.feat_lim : n.u.tok0 + r < n.u.tok_lim)
        n.lane_scale = p.row_scale[(COLS ? n.u.wrow0 : n.u.tok0) + r];
#pragma unroll
      for (int i = 0; i < kPartChunks; ++i) {
        // with COLS a warp takes every kParts-th chunk, so that short tiles spread over the warps
        const int c = (COLS ? (i * kParts + part) * 32 : part * kPartCols + i * 32) + lane;
        const bool in = COLS ? n.u.tok0 + c < n.u.tok_lim : n.u.feat0 + c < n.u.feat_lim;
        n.scale[i] = in ? p.col_scale[(COLS ? n.u.tok0 : n.u.wrow0) + c] : 0.f;
        n.bias[i] = has_bias(EPI) && in ? bf2f(p.bias[n.u.feat0 + c]) : 0.f;
      }
      return n;
    };
    Ahead next;
    if (pair < units) next = ahead(pair);
    int local = 0;
    for (int w = pair; w < units && !*abort_flag; w += pairs, ++local) {
      const Unit u = next.u;
      const float lane_scale = next.lane_scale;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kPartChunks; ++i) {
        cscale[i * 32 + lane] = next.scale[i];
        if (has_bias(EPI)) cbias[i * 32 + lane] = next.bias[i];
      }
      __syncwarp();
      if (w + pairs < units) next = ahead(w + pairs);
      const int acc = local & 1;
      const uint32_t freed = cluster_map(smem_u32(&tempty[acc]), 0);
      const uint32_t t0 = tmem_base + ((uint32_t)(q * 32) << 16) + acc * kPairTile;
      if (!mbar_wait(&tfull[acc], (local >> 1) & 1, p.err)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      if constexpr (COLS) {
        // 32 features a warp
        for (int c = part; c < u.n / 32; c += kParts) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t0 + c * 32, r);
          tmem_ld_wait();
          if (c + kParts >= u.n / 32) {  // all read: the accumulator is free for the tile after next
            tc_fence_before();
            __syncwarp();
            if (lane == 0) cluster_arrive_relaxed(freed);
          }
          emit_features<EPI, 32>(r, u.feat0 + rank * BM + q * 32, u.tok0 + c * 32, lane_scale, cscale + c / kParts * 32, u,
                                 lane, p);
        }
        if (part >= u.n / 32 && lane == 0) cluster_arrive_relaxed(freed);  // nothing of this tile is this warp's
      } else {
        // 32 token rows a warp
        const int64_t tok = u.tok0 + rank * BM + q * 32 + lane;
        const bool live = tok < u.tok_lim;
#pragma unroll
        for (int ch = 0; ch < kPartChunks; ++ch) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t0 + part * kPartCols + ch * 32, r);
          tmem_ld_wait();
          if (ch == kPartChunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) cluster_arrive_relaxed(freed);
          }
          if (live)
            emit_row<EPI>(r, tok, u.feat0 + part * kPartCols + ch * 32, lane_scale, cscale + ch * 32, cbias + ch * 32, wide, u,
                          p);
          __syncwarp();
        }
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // neither CTA leaves while the other may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kPairTile);
  }
}

// ---------------------------------------------------------------------------
// Few tokens per expert: one persistent CTA per SM walks the (expert, feature
// tile, token tile) units; the ring runs on across units and the accumulator
// is double-buffered.  Bound by the weights' bytes: 8 experts of 28672 x 4096 at
// 8 tokens each 146 us (6.4 TB/s, 98 % of the copy rate), 64 of 2816 x 2048 at 3
// tokens 59 us (94 %), 64 of 2048 x 1408 34.6 us (81 %; 6.9 tiles an SM).
// ---------------------------------------------------------------------------
template <int BN>
struct GroupCfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 200 * 1024 / STAGE_BYTES;
  static constexpr int TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*align*/ + 512 /*barriers*/ + 16 * BN /*token scales*/ + kGroupTabBytes;
  static constexpr uint32_t IDESC = idesc_i8_s32(BM, BN);
};

template <int BN, int EPI>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_i8_group_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
  using C = GroupCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* tscale = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + 512);  // of the tokens, per warp
  int* gtab = reinterpret_cast<int*>(tscale + 4 * BN);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 128);
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  pdl_wait();
  if (warp == 0) fill_group_table<BN>(gtab, p, lane);
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  const int units = gtab[2 * p.groups + 1];

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int w = blockIdx.x; w < units && !*abort_flag; w += gridDim.x) {
        const Unit u = group_unit<BN, BM>(w, p, gtab);
        for (int kb = 0; kb < p.kb_total; ++kb, ++issued) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.err)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
          tma_load_2d(sA + stage * C::A_BYTES, &tmA, &full[stage], kb * BK, u.wrow0);
          tma_load_2d(sB + stage * C::B_BYTES, &tmB, &full[stage], kb * BK, u.tok0);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (*abort_flag) drain_loads(full, C::STAGES, issued, p.err);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int w = blockIdx.x; w < units && !*abort_flag; w += gridDim.x, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, p.err)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        bool ok = true;
        for (int kb = 0; kb < p.kb_total; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * C::A_BYTES);
          const uint32_t b0 = smem_u32(sB + stage * C::B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_i8(tmem_base + acc * BN, smem_desc_k128(a0 + k * 32), smem_desc_k128(b0 + k * 32), C::IDESC,
                    (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        umma_commit(&tfull[acc]);
        if (!ok) {
          *abort_flag = 1;
          break;
        }
      }
      if (*abort_flag) {  // products in flight end before the operands' memory and TMEM go
        umma_commit(drained);
        mbar_wait(drained, 0, p.err);
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..5) ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    float* ts = tscale + q * BN;
    int local = 0;
    for (int w = blockIdx.x; w < units && !*abort_flag; w += gridDim.x, ++local) {
      const Unit u = group_unit<BN, BM>(w, p, gtab);
      const int acc = local & 1;
      const float fscale = u.feat0 + q * 32 + lane < u.feat_lim ? p.row_scale[u.wrow0 + q * 32 + lane] : 0.f;
      __syncwarp();
      for (int i = lane; i < BN; i += 32) ts[i] = u.tok0 + i < u.tok_lim ? p.col_scale[u.tok0 + i] : 0.f;
      __syncwarp();
      if (!mbar_wait(&tfull[acc], (local >> 1) & 1, p.err)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      constexpr int CW = BN < 32 ? BN : 32;
#pragma unroll 1
      for (int c = 0; c < BN && u.tok0 + c < u.tok_lim; c += CW) {
        uint32_t r[CW];
        const uint32_t t = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + c;
        if constexpr (CW == 32) tmem_ld_32x32b_x32(t, r);
        else tmem_ld_32x32b_x16(t, r);
        tmem_ld_wait();
        emit_features<EPI, CW>(r, u.feat0 + q * 32, u.tok0 + c, fscale, ts + c, u, lane, p);
      }
      tc_fence_before();
      mbar_arrive(&tempty[acc]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Few tokens: one tile of 128 features x BN tokens per cluster, its K range
// split over the cluster's CTAs; two CTAs per SM, so that one's epilogue runs
// under another's loads.  Bound by the weights' bytes and the ends of the launch:
// 64 x 24576 x 4096 with SwiGLU 20.9 us in a chain of launches (100.7 MB, 15.4 us
// at the copy rate: 1.3 us to the first tile, the stream done at 15 to 17, 2 for
// the last epilogue, 2 to the next launch), 64 x 6144 x 4096 9.6 us (floor 3.8),
// 1 x 4096 x 4096 6.2 us (2.6).  Asking for the weights' first tiles into L2 while
// the previous kernel drains gained nothing (20.8 / 21.0 / 21.6 us with 0 / 4 / 8
// k-blocks), and further ahead inside the loop it lost (18.5 to 22.5 us at one
// token).
// ---------------------------------------------------------------------------
template <int BN>
struct SplitCfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 100 * 1024 / STAGE_BYTES;  // two CTAs per SM
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/ + BN * 4 /*token scales*/;
  static constexpr uint32_t IDESC = idesc_i8_s32(BM, BN);
  static_assert(BN * BM * 4 <= STAGES * STAGE_BYTES, "the partial tile reuses the ring");
};

// Four consecutive features f0.. of token `tok`, values already scaled, through
// the epilogue with their bias and residual.
template <int EPI>
__device__ __forceinline__ void emit4(float v[4], const float bias[4], const float res[4], int64_t f0, int64_t tok,
                                      const Params& p) {
  if (EPI == B200_EPI_SWIGLU) {
    *reinterpret_cast<uint32_t*>(p.C + tok * p.ldc + f0 / 2) = pack2(silu_f(v[0]) * v[1], silu_f(v[2]) * v[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] += bias[i];
    if (EPI == B200_EPI_BIAS_GELU) v[i] = gelu_tanh_f(v[i]);
    v[i] += res[i];
  }
  *reinterpret_cast<uint2*>(p.C + tok * p.ldc + f0) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
}

// Tokens t0, t0 + 6, ... < last (of the tile that begins at tok0) of the lane's four features: the partial sums of
// the cluster's S <= NS CTAs added up and finished.  U tokens x NS loads are in
// flight at once.
template <int EPI, int U, int NS>
__device__ __forceinline__ void finish_tokens(uint32_t base, int S, int t0, int last, int64_t tok0, const float4& fs,
                                              const float fb[4], const float* tscale, int64_t f0, const Params& p) {
  constexpr int kWarps = kThreads / 32;
  for (; t0 < last; t0 += U * kWarps) {
    int4 a[U][NS];
    float r[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * kWarps;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        a[u][s] = t < last && s < S ? cluster_load4(cluster_map(base + t * (BM * 4), s)) : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[u][i] = 0.f;
      if (has_residual(EPI) && t < last) add4(r[u], p.R + (tok0 + t) * p.ldr + f0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * kWarps;
      if (t >= last) continue;
      int4 sum = a[u][0];
#pragma unroll
      for (int s = 1; s < NS; ++s)
        sum.x += a[u][s].x, sum.y += a[u][s].y, sum.z += a[u][s].z, sum.w += a[u][s].w;
      const float ts = tscale[t];
      float v[4] = {(float)sum.x * ts * fs.x, (float)sum.y * ts * fs.y, (float)sum.z * ts * fs.z, (float)sum.w * ts * fs.w};
      emit4<EPI>(v, fb, r[u], f0, tok0 + t, p);
    }
  }
}

template <int BN, int EPI>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_i8_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const Params p) {
  using C = SplitCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  int* part = reinterpret_cast<int*>(smem);  // [token][128 features], once the ring is drained
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  float* tscale = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE_BYTES + 256);  // of the tokens

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = (int)cluster_size(), rank = (int)cluster_rank();
  const int tile = (int)(blockIdx.x / S);
  const int row0 = tile % p.tiles_m * BM;
  const int tok0 = tile / p.tiles_m * BN;
  const int kb0 = rank * p.kb_per_split, nkb = min(p.kb_total - kb0, p.kb_per_split);
  const int tokens = min((int)p.cols - tok0, BN);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  __syncthreads();
  pdl_wait();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < nkb; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1, p.err)) {
          drain_loads(full, C::STAGES, i, p.err);
          break;
        }
        mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
        tma_load_2d(sA + stage * C::A_BYTES, &tmA, &full[stage], (kb0 + i) * BK, row0);
        tma_load_2d(sB + stage * C::B_BYTES, &tmB, &full[stage], (kb0 + i) * BK, tok0);
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else {
    // TMEM is allocated while the first tiles are on their way
    if (warp == 1) {
      tmem_alloc(tmem_slot, C::TMEM_COLS);
      tmem_relinquish();
      pdl_trigger();
    }
    tc_fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");  // warps 1-5
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (warp == 1) {
      // ---------------- MMA issuer ----------------
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; i < nkb; ++i) {
          if (!mbar_wait(&full[stage], phase, p.err)) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * C::A_BYTES);
          const uint32_t b0 = smem_u32(sB + stage * C::B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_i8(tmem_base, smem_desc_k128(a0 + k * 32), smem_desc_k128(b0 + k * 32), C::IDESC,
                    (i > 0 || k > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        umma_commit(tfull);  // after a wait that ran out, too: nothing is in flight once the epilogue has seen it
      }
      __syncwarp();
    } else {
      // ---------------- partial sums to shared memory (warps 2-5) ----------------
      const int q = warp & 3;  // TMEM lane quarter this warp may access
      const int rit = q * 32 + lane;
      if (rit < tokens) tscale[rit] = p.col_scale[tok0 + rit];
      const bool ok = mbar_wait(tfull, 0, p.err);
      tc_fence_after();
      constexpr int CW = BN < 32 ? BN : 32;
      for (int ch = 0; ch < BN / CW && ch * CW < tokens && ok; ++ch) {
        uint32_t r[CW];
        const uint32_t t = tmem_base + ((uint32_t)(q * 32) << 16) + ch * CW;
        if constexpr (CW == 32) tmem_ld_32x32b_x32(t, r);
        else tmem_ld_32x32b_x16(t, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < CW; ++i)
          if (ch * CW + i < tokens) part[(ch * CW + i) * BM + rit] = (int)r[i];
      }
      tc_fence_before();
      __syncwarp();
    }
    // TMEM goes back before this CTA waits for others of its cluster: no CTA
    // holds any while it waits for one that may still be asking for it
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
  }
  // This CTA finishes its share of the tokens: the cluster's partial sums
  // (integers: their order does not matter).  A lane keeps four features, a
  // warp takes every sixth token, and what does not depend on the sums is
  // loaded before they are there.
  const int share = (tokens + S - 1) / S;
  const int first = rank * share, last = min(tokens, first + share);
  const int64_t f0 = row0 + lane * 4;
  const bool live = f0 < p.rows;
  float4 fs = make_float4(0.f, 0.f, 0.f, 0.f);
  float fb[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    fs = *reinterpret_cast<const float4*>(p.row_scale + f0);
    if (has_bias(EPI)) add4(fb, p.bias + f0);
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  if (live) {
    const uint32_t base = smem_u32(part) + lane * 16;
    if (S == 1) finish_tokens<EPI, 4, 1>(base, S, first + warp, last, tok0, fs, fb, tscale, f0, p);
    else if (S <= 4) finish_tokens<EPI, 4, 4>(base, S, first + warp, last, tok0, fs, fb, tscale, f0, p);
    else finish_tokens<EPI, 2, 8>(base, S, first + warp, last, tok0, fs, fb, tscale, f0, p);
  }
  if (S > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}

// 2-D byte tensor map over a row-major [rows, K] matrix with row stride ld,
// box = box_rows x 128 bytes; what lies outside reads as zero.
bool make_tmap(CUtensorMap* m, const void* ptr, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  EncodeTiledFn f = encode_fn();
  if (!f) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

int num_sms() {
  static int n[64] = {0};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return 148;
  if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] > 0 ? n[dev] : 148;
}

template <typename Kernel>
bool allow_smem(Kernel k, int bytes, bool (&done)[64]) {
  const int dev = current_device();
  if (dev >= 0 && dev < 64 && done[dev]) return true;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev >= 0 && dev < 64) done[dev] = true;
  return true;
}

template <int EPI, int MODE>
int launch_pair(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int64_t units, cudaStream_t st) {
  auto k = gemm_i8_pair_kernel<EPI, MODE>;
  static bool done[64] = {false};
  if (!allow_smem(k, kPairSmem, done)) return B200_ERROR_UNSUPPORTED;
  const int pairs = (int)std::min<int64_t>(units, num_sms() / 2);
  launch_clusters(k, 2, dim3(2 * pairs), kPairThreads, kPairSmem, st, a, b, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

template <int BN, int EPI>
int launch_split(const CUtensorMap& tok, const CUtensorMap& w, const Params& p, int splits, cudaStream_t st) {
  auto k = gemm_i8_split_kernel<BN, EPI>;
  static bool done[64] = {false};
  if (!allow_smem(k, SplitCfg<BN>::SMEM, done)) return B200_ERROR_UNSUPPORTED;
  launch_clusters(k, splits, dim3(p.tiles_m * p.tiles_n * splits), kThreads, SplitCfg<BN>::SMEM, st, w, tok, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

template <int BN, int EPI>
int launch_group(const CUtensorMap& tok, const CUtensorMap& w, const Params& p, int64_t units, cudaStream_t st) {
  auto k = gemm_i8_group_kernel<BN, EPI>;
  static bool done[64] = {false};
  if (!allow_smem(k, GroupCfg<BN>::SMEM, done)) return B200_ERROR_UNSUPPORTED;
  launch_kernel(k, dim3((unsigned)std::min<int64_t>(units, num_sms())), kThreads, GroupCfg<BN>::SMEM, st, w, tok, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

// form: the token tile of the single-CTA form, or one of the pairs' two.
constexpr int kFormCols = 0, kFormRows = 1;
template <int EPI>
int launch_grouped(int form, const CUtensorMap& tok, const CUtensorMap& w, const Params& p, int64_t units, cudaStream_t st) {
  switch (form) {
    case 16: return launch_group<16, EPI>(tok, w, p, units, st);
    case 32: return launch_group<32, EPI>(tok, w, p, units, st);
    case 64: return launch_group<64, EPI>(tok, w, p, units, st);
    case kFormCols: return launch_pair<EPI, kCols>(w, tok, p, units, st);
    default: return launch_pair<EPI, kRows>(tok, w, p, units, st);
  }
}

// bn: the token tile of the split form, 0 for CTA pairs.
template <int EPI>
int launch_plain(int bn, int splits, const CUtensorMap& tok, const CUtensorMap& w, const Params& p, cudaStream_t st) {
  switch (bn) {
    case 16: return launch_split<16, EPI>(tok, w, p, splits, st);
    case 32: return launch_split<32, EPI>(tok, w, p, splits, st);
    case 64: return launch_split<64, EPI>(tok, w, p, splits, st);
    case 128: return launch_split<128, EPI>(tok, w, p, splits, st);
    default: return launch_pair<EPI, kPlain>(tok, w, p, (int64_t)p.tiles_m * p.tiles_n, st);
  }
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// CTAs of a cluster that share one 128-feature tile's K range: as many as keep
// two k-blocks each and fit one wave of clusters (256 of the 296 places: a
// cluster needs its places within one group of SMs, and 288 CTAs of 48 tiles
// already take two waves, 13.7 us against 9.6 at 192).  Past 4 the exchange
// costs more than a short K gains (4096 x 4096, one token: 6.2 us at 4, 6.9 at
// 8) and less than a long one does (12288: 12.6 at 4, 11.5 at 8).
int plan_splits(int tiles, int kb_total) {
  const int most = kb_total >= 64 ? 8 : 4;
  int s = 1;
  while (s < most && tiles * (s + 1) <= 256 && kb_total / (s + 1) >= 2) ++s;
  return s;
}

// CTA pairs once their 256 x 256 tiles keep five eighths of them busy (a narrow
// M or N would waste the tile), us split / pairs: 512 x 6144 x 4096 (48 tiles)
// 18.2 / 17.3, 512 x 4096 x 4096 (32) 14.8 / 18.6, 777 x 4096 x 1024 (64) 11.7 /
// 10.7, 2048 x 4096 x 4096 (128) 41 / 31, 1024 x 24576 x 4096 (384) 132 / 75.
bool use_pairs(int64_t M, int64_t N, int sms) {
  const int64_t tiles = ((M + kPairTile - 1) / kPairTile) * ((N + kPairTile - 1) / kPairTile);
  return M > 128 && N > 128 && tiles * 8 >= sms / 2 * 5;
}

// The checks that the plain and the grouped call share.
bool operands_ok(const void* A, int64_t lda, const void* as, const void* B, int64_t ldb, const void* bs, const void* C,
                 int64_t ldc, int64_t N, int64_t K, int epi) {
  if (!A || !as || !B || !bs || !C || N < 0 || K <= 0 || K % 16 || lda % 16 || ldb % 16 || lda < K || ldb < K ||
      ldc % 8 || N % (epi == B200_EPI_SWIGLU ? 16 : 8) || ldc < (epi == B200_EPI_SWIGLU ? N / 2 : N))
    return false;
  return aligned(A, 16) && aligned(B, 16) && aligned(C, 16) && aligned(as, 16) && aligned(bs, 16);
}

}  // namespace

extern "C" int b200_gemm_int8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B, int64_t ldb,
                              const float* b_scale, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                              int epilogue, const void* bias, const void* residual, int64_t ldr,
                              b200_stream_t stream) {
  if (epilogue < B200_EPI_NONE || epilogue > B200_EPI_BIAS_RESIDUAL || M < 0) return B200_ERROR_INVALID_PARAM;
  if (!operands_ok(A, lda, a_scale, B, ldb, b_scale, C, ldc, N, K, epilogue)) return B200_ERROR_INVALID_PARAM;
  if (has_bias(epilogue) && (!bias || !aligned(bias, 16))) return B200_ERROR_INVALID_PARAM;
  if (has_residual(epilogue) && (!residual || !aligned(residual, 16) || ldr % 8 || ldr < N))
    return B200_ERROR_INVALID_PARAM;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2 || K > kMaxK) return B200_ERROR_UNSUPPORTED;
  if (M == 0 || N == 0) return B200_OK;
  Params p{};
  p.kb_total = (int)((K + BK - 1) / BK);
  p.C = static_cast<__nv_bfloat16*>(C);
  p.ldc = ldc;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.R = static_cast<const __nv_bfloat16*>(residual);
  p.ldr = ldr;
  p.err = b200::error_word(current_device());
  const auto tiles = [](int64_t n, int64_t t) { return (n + t - 1) / t; };
  const bool pairs = use_pairs(M, N, num_sms());
  const int bn = pairs ? 0 : (M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128);
  int splits = 1;
  if (pairs) {
    p.rows = M;
    p.cols = N;
    p.tiles_m = (int)tiles(M, kPairTile);
    p.tiles_n = (int)tiles(N, kPairTile);
    p.row_scale = a_scale;
    p.col_scale = b_scale;
  } else {
    p.rows = N;
    p.cols = M;
    p.tiles_m = (int)tiles(N, BM);
    p.tiles_n = (int)tiles(M, bn);
    p.row_scale = b_scale;
    p.col_scale = a_scale;
  }
  if ((int64_t)p.tiles_m * p.tiles_n > INT32_MAX / 16) return B200_ERROR_UNSUPPORTED;
  if (!pairs) {
    splits = plan_splits(p.tiles_m * p.tiles_n, p.kb_total);
    p.kb_per_split = (int)tiles(p.kb_total, splits);
    splits = (int)tiles(p.kb_total, p.kb_per_split);
  }
  CUtensorMap tok, w;
  if (!make_tmap(&tok, A, M, K, lda, pairs ? BM : bn) || !make_tmap(&w, B, N, K, ldb, BM)) return B200_ERROR_UNSUPPORTED;
  switch (epilogue) {
    case B200_EPI_NONE: return launch_plain<B200_EPI_NONE>(bn, splits, tok, w, p, stream);
    case B200_EPI_BIAS: return launch_plain<B200_EPI_BIAS>(bn, splits, tok, w, p, stream);
    case B200_EPI_RESIDUAL: return launch_plain<B200_EPI_RESIDUAL>(bn, splits, tok, w, p, stream);
    case B200_EPI_SWIGLU: return launch_plain<B200_EPI_SWIGLU>(bn, splits, tok, w, p, stream);
    case B200_EPI_BIAS_GELU: return launch_plain<B200_EPI_BIAS_GELU>(bn, splits, tok, w, p, stream);
    default: return launch_plain<B200_EPI_BIAS_RESIDUAL>(bn, splits, tok, w, p, stream);
  }
}

extern "C" int b200_grouped_gemm_int8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B, int64_t ldb,
                                      const float* b_scale, void* C, int64_t ldc, const int32_t* group_offsets,
                                      int groups, int64_t rows, int64_t N, int64_t K, int epilogue,
                                      b200_stream_t stream) {
  if (epilogue != B200_EPI_NONE && epilogue != B200_EPI_SWIGLU) return B200_ERROR_INVALID_PARAM;
  if (!group_offsets || !aligned(group_offsets, 4) || groups <= 0 || groups > kMaxGroups || rows < 0 || N <= 0)
    return B200_ERROR_INVALID_PARAM;
  if (!operands_ok(A, lda, a_scale, B, ldb, b_scale, C, ldc, N, K, epilogue)) return B200_ERROR_INVALID_PARAM;
  if (rows > INT32_MAX / 4 || N > INT32_MAX / 4 || groups * N > INT32_MAX / 4 || K > kMaxK)
    return B200_ERROR_UNSUPPORTED;
  if (rows == 0) return B200_OK;
  // By the average tokens of a group: up to 56, single CTAs with weights on the
  // 128-row side and up to bn tokens on the N side (bn leaves room for a group of
  // twice the average, past which its weights are read, from L2, again); up to
  // 160, pairs with the tokens on the N side; beyond, pairs with the tokens on
  // the M side, whose epilogue costs the main loop less.  64 groups of 2816 x
  // 2048 with SwiGLU, us: at 48 tokens 65 / 72 / -, at 64 79 / 74 / 82, at 128
  // 128 / 80 / 84, at 192 - / 88 / 87, at 768 - / 276 / 258.
  const bool few = rows <= 56LL * groups, cols = !few && rows <= 160LL * groups;
  const int bn = rows <= 8LL * groups ? 16 : rows <= 16LL * groups ? 32 : 64;
  const int feat_tile = few ? BM : kPairTile, tok_tile = few ? bn : kPairTile;
  Params p{};
  p.kb_total = (int)((K + BK - 1) / BK);
  p.row_scale = few || cols ? b_scale : a_scale;
  p.col_scale = few || cols ? a_scale : b_scale;
  p.C = static_cast<__nv_bfloat16*>(C);
  p.ldc = ldc;
  p.err = b200::error_word(current_device());
  p.goff = group_offsets;
  p.groups = groups;
  p.gN = N;
  p.gF = (int)((N + feat_tile - 1) / feat_tile);
  p.gRows = rows;
  // host upper bound of the units: every group's partial token tile + the full ones
  const int64_t max_units = ((rows + tok_tile - 1) / tok_tile + groups) * (int64_t)p.gF;
  if (max_units > INT32_MAX / 2) return B200_ERROR_UNSUPPORTED;
  CUtensorMap w, tok;
  if (!make_tmap(&w, B, (int64_t)groups * N, K, ldb, BM) ||
      !make_tmap(&tok, A, rows, K, lda, few ? bn : cols ? kTokBox : BM))
    return B200_ERROR_UNSUPPORTED;
  const int form = few ? bn : cols ? kFormCols : kFormRows;
  return epilogue == B200_EPI_SWIGLU ? launch_grouped<B200_EPI_SWIGLU>(form, tok, w, p, max_units, stream)
                                     : launch_grouped<B200_EPI_NONE>(form, tok, w, p, max_units, stream);
}

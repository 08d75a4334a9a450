// 8-bit integer GEMM on the 5th-generation tensor cores:
//   C[m, n] = epi(a_scale[m] * b_scale[n] * sum_k A[m, k] B[n, k])
// with int8 operands, exact 32-bit integer sums and one rounding to bf16.
//
// One persistent CTA per SM, 192 threads:
//   warp 0      TMA producer: 128 x 128-byte tile of the row operand and
//               BN x 128-byte tile of the column operand per stage, 128-byte
//               swizzle, a ring of shared-memory stages.
//   warp 1      allocates TMEM; one thread issues tcgen05.mma kind::i8
//               (M = 128, N = BN, K = 32) into one of two TMEM accumulators.
//   warps 2-5   epilogue: tcgen05.ld, scales, bias / residual / SwiGLU / GELU,
//               bf16 stores.
// Few token rows run "swapped": the weights feed the 128-row side, the tokens
// the N side, and the epilogue writes the transpose.
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
constexpr int kGroupM = 16;
constexpr int kMaxGroups = 256;                           // experts of one grouped GEMM
constexpr int kGroupTabBytes = 2 * (kMaxGroups + 2) * 4;  // row offsets + unit prefix in shared memory
// The largest |sum| is 128 * 128 * K (both operands may hold -128): it fits 31 bits up to here.
constexpr int64_t kMaxK = 131056;

template <int BN>
struct Cfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 200 * 1024 / STAGE_BYTES;
  static constexpr int TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*align*/ + 512 /*barriers*/ + kGroupTabBytes;
  static constexpr uint32_t IDESC = idesc_i8_s32(BM, BN);
};

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
  int a_row, b_row;         // TMA rows of both operands
  int64_t row0, col0;       // output origin (token / feature by orientation)
  int64_t row_lim, col_lim;
  int64_t rs0, cs0;         // scale index of row0 / col0
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

template <int BN, bool SWAP, bool GROUPED>
__device__ __forceinline__ Unit get_unit(int w, const Params& p, const int* gtab) {
  Unit u;
  if (!GROUPED) {
    const int group = kGroupM * p.tiles_n;
    const int first_m = w / group * kGroupM;
    const int gm = min(p.tiles_m - first_m, kGroupM);
    const int r = w % group;
    const int tm = first_m + r % gm, tn = r / gm;
    u.a_row = tm * BM;
    u.b_row = tn * BN;
    u.row0 = u.rs0 = u.a_row;
    u.col0 = u.cs0 = u.b_row;
    u.row_lim = p.rows;
    u.col_lim = p.cols;
    return u;
  }
  const int* up = gtab + p.groups + 1;
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (up[mid] <= w) lo = mid;
    else hi = mid;
  }
  const int g = lo;
  constexpr int TOKT = SWAP ? BN : BM, FEATT = SWAP ? BM : BN;
  const int t0 = gtab[g], t1 = gtab[g + 1];
  const int tt = (t1 - t0 + TOKT - 1) / TOKT;
  const int r = w - up[g];
  const int tok = t0 + r % tt * TOKT, feat = r / tt * FEATT;
  const int wrow = (int)(g * p.gN) + feat;
  if (SWAP) {
    u.a_row = wrow;
    u.b_row = tok;
    u.row0 = feat;
    u.rs0 = wrow;
    u.row_lim = p.gN;
    u.col0 = u.cs0 = tok;
    u.col_lim = t1;
  } else {
    u.a_row = tok;
    u.b_row = wrow;
    u.row0 = u.rs0 = tok;
    u.row_lim = t1;
    u.col0 = feat;
    u.cs0 = wrow;
    u.col_lim = p.gN;
  }
  return u;
}

// Store CW accumulator columns of one MMA row with the epilogue.  Normal
// orientation: the row is a token, the columns are features (vector stores).
// Swapped: the row is a feature (consecutive features in consecutive lanes),
// the columns are tokens.
template <int EPI, bool SWAP, int CW>
__device__ __forceinline__ void emit_chunk(const uint32_t acc[CW], int64_t row, int64_t col0, float rscale,
                                           const float* cscale, const Unit& u, int lane, const Params& p) {
  float v[CW];
#pragma unroll
  for (int i = 0; i < CW; ++i) v[i] = (float)(int)acc[i] * rscale;
  if (!SWAP) {
    if (row >= u.row_lim) return;
#pragma unroll
    for (int g = 0; g < CW / 8; ++g) {
      const int64_t c = col0 + g * 8;
      if (c >= u.col_lim) continue;
      float* x = v + 8 * g;
      const float4 s0 = *reinterpret_cast<const float4*>(cscale + g * 8);
      const float4 s1 = *reinterpret_cast<const float4*>(cscale + g * 8 + 4);
      x[0] *= s0.x, x[1] *= s0.y, x[2] *= s0.z, x[3] *= s0.w;
      x[4] *= s1.x, x[5] *= s1.y, x[6] *= s1.z, x[7] *= s1.w;
      if (has_bias(EPI)) {
        float b[8];
        unpack8(*reinterpret_cast<const uint4*>(p.bias + c), b);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += b[i];
      }
      if (EPI == B200_EPI_BIAS_GELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = gelu_tanh_f(x[i]);
      }
      if (has_residual(EPI)) {
        float r[8];
        unpack8(*reinterpret_cast<const uint4*>(p.R + row * p.ldr + c), r);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += r[i];
      }
      if (EPI == B200_EPI_SWIGLU) {
        uint2 o;
        o.x = pack2(silu_f(x[0]) * x[1], silu_f(x[2]) * x[3]);
        o.y = pack2(silu_f(x[4]) * x[5], silu_f(x[6]) * x[7]);
        *reinterpret_cast<uint2*>(p.C + row * p.ldc + c / 2) = o;
      } else {
        *reinterpret_cast<uint4*>(p.C + row * p.ldc + c) = pack8(x);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < CW; ++i) v[i] *= col0 + i < u.col_lim ? cscale[i] : 0.f;
  if (EPI == B200_EPI_SWIGLU) {
    // lanes 2j / 2j+1 hold the gate / up rows of feature j: the even lane
    // finishes the first half of the chunk's tokens, the odd lane the second
    const bool odd = lane & 1;
    const int64_t f = row >> 1;
    constexpr int H = CW / 2;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[H + i], 1);
      const int64_t tok = col0 + (odd ? H + i : i);
      const float o = odd ? silu_f(other) * v[H + i] : silu_f(v[i]) * other;
      if (row < u.row_lim && tok < u.col_lim) p.C[tok * p.ldc + f] = f2bf(o);
    }
    return;
  }
  if (row >= u.row_lim) return;
  const float b = has_bias(EPI) ? bf2f(p.bias[row]) : 0.f;
#pragma unroll
  for (int i = 0; i < CW; ++i) {
    const int64_t tok = col0 + i;
    if (tok >= u.col_lim) continue;
    float x = v[i] + b;
    if (EPI == B200_EPI_BIAS_GELU) x = gelu_tanh_f(x);
    if (has_residual(EPI)) x += bf2f(p.R[tok * p.ldr + row]);
    p.C[tok * p.ldc + row] = f2bf(x);
  }
}

template <int BN, int EPI, bool SWAP, bool GROUPED>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* gtab = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE_BYTES + 512);  // grouped launches only

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int units = p.tiles_m * p.tiles_n;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 128);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  pdl_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  if (GROUPED) {
    if (threadIdx.x == 0) {
      int prev = 0, run = 0;
      for (int g = 0; g <= p.groups; ++g) {
        int v = p.goff[g];
        if (v < prev || v > p.gRows || (g == 0 && v != 0)) {
          raise_error(p.err, DEV_ERR_BAD_INDEX);
          v = min(max(v, prev), (int)p.gRows);
          if (g == 0) v = 0;
        }
        gtab[g] = prev = v;
      }
      constexpr int TOKT = SWAP ? BN : BM;
      for (int g = 0; g < p.groups; ++g) {
        gtab[p.groups + 1 + g] = run;
        run += ((gtab[g + 1] - gtab[g] + TOKT - 1) / TOKT) * p.gF;
      }
      gtab[2 * p.groups + 1] = run;
    }
    __syncthreads();
    units = gtab[2 * p.groups + 1];
  }

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int w = blockIdx.x; w < units && !*abort_flag; w += gridDim.x) {
        const Unit u = get_unit<BN, SWAP, GROUPED>(w, p, gtab);
        for (int kb = 0; kb < p.kb_total; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.err)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
          tma_load_2d(sA + stage * C::A_BYTES, &tmA, &full[stage], kb * BK, u.a_row);
          tma_load_2d(sB + stage * C::B_BYTES, &tmB, &full[stage], kb * BK, u.b_row);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
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
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..5) ----------------
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const int rit = q * 32 + lane;
    constexpr int CW = BN < 32 ? BN : 32;
    int local = 0;
    for (int w = blockIdx.x; w < units && !*abort_flag; w += gridDim.x, ++local) {
      const Unit u = get_unit<BN, SWAP, GROUPED>(w, p, gtab);
      const int acc = local & 1;
      const int64_t row = u.row0 + rit;
      const float rscale = row < u.row_lim ? p.row_scale[u.rs0 + rit] : 0.f;
      if (!mbar_wait(&tfull[acc], (local >> 1) & 1, p.err)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int ch = 0; ch < BN / CW; ++ch) {
        uint32_t r[CW];
        const uint32_t t = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + ch * CW;
        if constexpr (CW == 32) tmem_ld_32x32b_x32(t, r);
        else tmem_ld_32x32b_x16(t, r);
        tmem_ld_wait();
        emit_chunk<EPI, SWAP, CW>(r, row, u.col0 + ch * CW, rscale, p.col_scale + u.cs0 + ch * CW, u, lane, p);
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
// Few tokens (M <= 128): one 128-feature tile per cluster, its K range split
// over the cluster's CTAs.
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

__device__ __forceinline__ void add4(float v[4], const __nv_bfloat16* src) {
  const uint2 u = *reinterpret_cast<const uint2*>(src);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  v[0] += a.x, v[1] += a.y, v[2] += b.x, v[3] += b.y;
}

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

// Tokens t0, t0 + 6, ... < last of the lane's four features: the partial sums of
// the cluster's S <= NS CTAs added up and finished.  U tokens x NS loads are in
// flight at once.
template <int EPI, int U, int NS>
__device__ __forceinline__ void finish_tokens(uint32_t base, int S, int t0, int last, const float4& fs, const float fb[4],
                                              const float* tscale, int64_t f0, const Params& p) {
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
      if (has_residual(EPI) && t < last) add4(r[u], p.R + (int64_t)t * p.ldr + f0);
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
      emit4<EPI>(v, fb, r[u], f0, t, p);
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
  const int row0 = (int)(blockIdx.x / S) * BM;
  const int kb0 = rank * p.kb_per_split, nkb = min(p.kb_total - kb0, p.kb_per_split);
  const int tokens = (int)p.cols;

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
        if (!mbar_wait(&empty[stage], phase ^ 1, p.err)) break;
        mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
        tma_load_2d(sA + stage * C::A_BYTES, &tmA, &full[stage], (kb0 + i) * BK, row0);
        tma_load_2d(sB + stage * C::B_BYTES, &tmB, &full[stage], (kb0 + i) * BK, 0);
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
        umma_commit(tfull);
      }
      __syncwarp();
    } else {
      // ---------------- partial sums to shared memory (warps 2-5) ----------------
      const int q = warp & 3;  // TMEM lane quarter this warp may access
      const int rit = q * 32 + lane;
      if (rit < tokens) tscale[rit] = p.col_scale[rit];
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
    if (S == 1) finish_tokens<EPI, 4, 1>(base, S, first + warp, last, fs, fb, tscale, f0, p);
    else if (S <= 4) finish_tokens<EPI, 4, 4>(base, S, first + warp, last, fs, fb, tscale, f0, p);
    else finish_tokens<EPI, 2, 8>(base, S, first + warp, last, fs, fb, tscale, f0, p);
  }
  __syncwarp();
  if (S > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, C::TMEM_COLS);
  }
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

template <int BN, int EPI, bool SWAP, bool GROUPED>
int launch_t(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t st) {
  auto k = gemm_i8_kernel<BN, EPI, SWAP, GROUPED>;
  static bool attr_set[64] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::SMEM) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  launch_kernel(k, dim3(grid), kThreads, Cfg<BN>::SMEM, st, a, b, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

template <int BN>
int launch_epi(int epi, const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t st) {
  switch (epi) {
    case B200_EPI_NONE: return launch_t<BN, B200_EPI_NONE, false, false>(a, b, p, grid, st);
    case B200_EPI_BIAS: return launch_t<BN, B200_EPI_BIAS, false, false>(a, b, p, grid, st);
    case B200_EPI_RESIDUAL: return launch_t<BN, B200_EPI_RESIDUAL, false, false>(a, b, p, grid, st);
    case B200_EPI_SWIGLU: return launch_t<BN, B200_EPI_SWIGLU, false, false>(a, b, p, grid, st);
    case B200_EPI_BIAS_GELU: return launch_t<BN, B200_EPI_BIAS_GELU, false, false>(a, b, p, grid, st);
    case B200_EPI_BIAS_RESIDUAL: return launch_t<BN, B200_EPI_BIAS_RESIDUAL, false, false>(a, b, p, grid, st);
  }
  return B200_ERROR_INVALID_PARAM;
}

template <int BN, int EPI>
int launch_split_t(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int splits, cudaStream_t st) {
  auto k = gemm_i8_split_kernel<BN, EPI>;
  static bool attr_set[64] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitCfg<BN>::SMEM) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  launch_clusters(k, splits, dim3(p.tiles_m * splits), kThreads, SplitCfg<BN>::SMEM, st, a, b, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

template <int BN>
int launch_split(int epi, const CUtensorMap& a, const CUtensorMap& b, const Params& p, int splits, cudaStream_t st) {
  switch (epi) {
    case B200_EPI_NONE: return launch_split_t<BN, B200_EPI_NONE>(a, b, p, splits, st);
    case B200_EPI_BIAS: return launch_split_t<BN, B200_EPI_BIAS>(a, b, p, splits, st);
    case B200_EPI_RESIDUAL: return launch_split_t<BN, B200_EPI_RESIDUAL>(a, b, p, splits, st);
    case B200_EPI_SWIGLU: return launch_split_t<BN, B200_EPI_SWIGLU>(a, b, p, splits, st);
    case B200_EPI_BIAS_GELU: return launch_split_t<BN, B200_EPI_BIAS_GELU>(a, b, p, splits, st);
    case B200_EPI_BIAS_RESIDUAL: return launch_split_t<BN, B200_EPI_BIAS_RESIDUAL>(a, b, p, splits, st);
  }
  return B200_ERROR_INVALID_PARAM;
}

template <int BN, bool SWAP>
int launch_grouped(int epi, const CUtensorMap& a, const CUtensorMap& b, const Params& p, int grid, cudaStream_t st) {
  return epi == B200_EPI_SWIGLU ? launch_t<BN, B200_EPI_SWIGLU, SWAP, true>(a, b, p, grid, st)
                                : launch_t<BN, B200_EPI_NONE, SWAP, true>(a, b, p, grid, st);
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
  const bool swap = M <= 128;
  const int bn = swap ? (M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128) : (N > 128 ? 256 : 128);
  Params p{};
  p.rows = swap ? N : M;
  p.cols = swap ? M : N;
  p.tiles_m = (int)((p.rows + BM - 1) / BM);
  p.tiles_n = (int)((p.cols + bn - 1) / bn);
  p.kb_total = (int)((K + BK - 1) / BK);
  p.row_scale = swap ? b_scale : a_scale;
  p.col_scale = swap ? a_scale : b_scale;
  p.C = static_cast<__nv_bfloat16*>(C);
  p.ldc = ldc;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.R = static_cast<const __nv_bfloat16*>(residual);
  p.ldr = ldr;
  p.err = b200::error_word(current_device());
  if ((int64_t)p.tiles_m * p.tiles_n > INT32_MAX / 2) return B200_ERROR_UNSUPPORTED;
  CUtensorMap ta, tb;
  if (!make_tmap(&ta, swap ? B : A, p.rows, K, swap ? ldb : lda, BM) ||
      !make_tmap(&tb, swap ? A : B, p.cols, K, swap ? lda : ldb, bn))
    return B200_ERROR_UNSUPPORTED;
  if (swap) {
    const int splits = plan_splits(p.tiles_m, p.kb_total);
    p.kb_per_split = (p.kb_total + splits - 1) / splits;
    const int used = (p.kb_total + p.kb_per_split - 1) / p.kb_per_split;
    if (bn == 16) return launch_split<16>(epilogue, ta, tb, p, used, stream);
    if (bn == 32) return launch_split<32>(epilogue, ta, tb, p, used, stream);
    if (bn == 64) return launch_split<64>(epilogue, ta, tb, p, used, stream);
    return launch_split<128>(epilogue, ta, tb, p, used, stream);
  }
  const int grid = std::min(p.tiles_m * p.tiles_n, num_sms());
  return bn == 256 ? launch_epi<256>(epilogue, ta, tb, p, grid, stream)
                   : launch_epi<128>(epilogue, ta, tb, p, grid, stream);
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
  // Few tokens per group (decode): weights on the 128-row side, otherwise tokens.
  const bool swap = rows <= 96LL * groups;
  const int bn = swap ? 64 : (N > 128 ? 256 : 128);
  const int feat_tile = swap ? BM : bn, tok_tile = swap ? bn : BM;
  Params p{};
  p.kb_total = (int)((K + BK - 1) / BK);
  p.row_scale = swap ? b_scale : a_scale;
  p.col_scale = swap ? a_scale : b_scale;
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
  CUtensorMap tw, tt;
  if (!make_tmap(&tw, B, (int64_t)groups * N, K, ldb, feat_tile) || !make_tmap(&tt, A, rows, K, lda, tok_tile))
    return B200_ERROR_UNSUPPORTED;
  const int grid = (int)std::min<int64_t>(max_units, num_sms());
  if (swap) return launch_grouped<64, true>(epilogue, tw, tt, p, grid, stream);
  return bn == 256 ? launch_grouped<256, false>(epilogue, tt, tw, p, grid, stream)
                   : launch_grouped<128, false>(epilogue, tt, tw, p, grid, stream);
}

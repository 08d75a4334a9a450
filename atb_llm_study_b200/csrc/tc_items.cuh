// Attention of pairs of query tiles over lists of key tiles on the tcgen05
// tensor cores: the kernel of sliding-window prompts and of shared prefixes.
//
//   out = sum_j p_j v_j / sum_j p_j, p_j = 2^(q.k_j scale log2(e) - m)
//
// An item is one or two tiles of 128 query rows ("sides") that walk one list of
// 128-key tiles; a persistent CTA per SM walks its items.  Its warps:
//   0       TMA: each item's Q tiles, then K and V tiles through rings
//   1, 11   each issues the MMAs of a side.  Per key tile: O += P V of
//           the tile whose P is ready, right behind it S = Q K^T of the next tile
//           (the next item's first at an item's end).  Both sides use a K / V tile
//           while it is in shared memory.
//   2       looks through V tiles for NaN and infinities (below)
//   3-10    softmax, four warps a side, a thread a row: scores from TMEM, masked,
//           maximum, exponentials, sum, P as bf16 pairs over the scores, where the
//           MMA reads it.
// What a side's chain has to wait for itself (scores, softmax, P V) the other
// side's fills: the tensor core works for one while the softmax units work for
// the other.  At 128-wide heads a side's tile takes 1024 cycles of MMAs and as
// many of exponentials (16 a cycle and SM), so the two halves of the SM are
// equally loaded.  TMEM: two score tiles and two output accumulators, 4 x 128
// columns.  S of a side's next tile overwrites P that the P V before it reads: MMAs
// of one lane run in the order of their issue.
//
// The running maximum moves only when it grows by more than 2^8 (the rows of O
// in TMEM are then rescaled by their threads, seldom), which changes nothing in
// exact arithmetic and keeps P below 2^8 of its usual scale.
//
// Values that nobody sees must not reach anybody: P is 0 there, but 0 x NaN is
// not.  So the value rows of every tile that a side does not see as a whole (a
// prompt's end, its diagonal, the ends of the window and the sinks, a cache
// block's rest) are looked through, and those with a NaN or an infinity zeroed.
// A row that does see such a key gets NaN: the item's list of zeroed keys is
// looked through when its rows are stored.  (One warp takes 2000 cycles a tile,
// as long as V arrives ahead of its use; four were no faster in all.)
//
// P provides: HDK, HDV; Item with int n (key tiles, > 0), bool both (side 1 is
// there); Cursor(p) with bool next(Item&, err); load_q(p, item, side, ..) and
// load_k / load_v(p, item, tile, smem, map, bar, err): arrive on bar expecting
// bytes, copy; int key0(item, tile): its first key; bool whole(item, side, key):
// every row of the side sees the 128 keys from key on; visible(item, side, row,
// key): bits of the 32 from key on that a row sees; store(p, item, side, row, m, l, tO).
#pragma once

#include "tc_attention.cuh"

namespace {

constexpr int kSides = 2;
constexpr int kItemThreads = 384, kMma1Warp = 11;  // the second side's issuer
constexpr uint32_t kSideS = 0, kSideO = 256;  // TMEM columns of side 0's scores and outputs; side 1's lie 128 further
constexpr int kMaxEdgeTiles = 6;

struct Hidden {  // zeroed value rows of one item's edge tiles
  int any, count;
  int key0[kMaxEdgeTiles];
  uint32_t keys[kMaxEdgeTiles][4];
};

// sum += 0 x v, two bf16 values at once
B200_DEV void add_times_0(uint32_t& sum, uint32_t v) {
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(v), "r"(0u));
}

// Zeroes those of the 32 rows of a V tile from sV on that hold a NaN or an infinity; their bits.  One warp.
template <int BOXES>
B200_DEV uint32_t clear_nonfinite(uint8_t* sV) {
  const int lane = threadIdx.x & 31;
  // an instruction covers 4 rows, 8 lanes of 16 bytes a row (a row is 128 contiguous bytes of each box, whatever the
  // swizzle)
  uint4 v[BOXES * 8];
#pragma unroll
  for (int i = 0; i < BOXES * 8; ++i)
    v[i] = *reinterpret_cast<const uint4*>(sV + (i >> 3) * kBoxBytes + (i & 7) * 512 + lane * 16);
  // the sum of all values times 0 is 0 without one, and NaN with one
  uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < BOXES * 8; ++i) {
    add_times_0(sum[0], v[i].x);
    add_times_0(sum[1], v[i].y);
    add_times_0(sum[2], v[i].z);
    add_times_0(sum[3], v[i].w);
  }
  if (!__any_sync(0xffffffffu, ((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0)) return 0;
  uint32_t found = 0;
#pragma unroll 1
  for (int i = 0; i < BOXES * 8; ++i) {
    const uint4 u = *reinterpret_cast<const uint4*>(sV + (i >> 3) * kBoxBytes + (i & 7) * 512 + lane * 16);
    uint32_t s = 0;
    add_times_0(s, u.x);
    add_times_0(s, u.y);
    add_times_0(s, u.z);
    add_times_0(s, u.w);
    const uint32_t lanes = __ballot_sync(0xffffffffu, (s & 0x7fff7fffu) != 0);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (lanes & (0xffu << (8 * r))) found |= 1u << ((i & 7) * 4 + r);
  }
#pragma unroll 1
  for (uint32_t left = found; left; left &= left - 1) {
    const int r = __ffs(left) - 1;
    for (int c = lane; c < BOXES * 8; c += 32)
      *reinterpret_cast<uint4*>(sV + (c >> 3) * kBoxBytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor core reads the tile
  __syncwarp();
  return found;
}

// Bits [a, b) of 32.
B200_DEV uint32_t bit_range(int a, int b) {
  a = max(a, 0);
  b = min(b, 32);
  return b > a ? (0xffffffffu >> (32 - b + a)) << a : 0u;
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t r[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// max(a, b, c), NaN where one is
B200_DEV float fmax3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// m4 = maxima of four chains over 32 more raw scores (two an instruction); NaN stays.
B200_DEV void row_max(const uint32_t r[32], float m4[4]) {
#pragma unroll
  for (int c = 0; c < 16; ++c) m4[c & 3] = fmax3_nan(m4[c & 3], __uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
}

// Two floats an instruction.
B200_DEV uint64_t pair64(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
B200_DEV void unpair64(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
B200_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
B200_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two values without the special-function unit: x = n + f with n the
// nearest integer (adding 1.5 x 2^23 leaves it in the low bits) and |f| <= 1/2;
// 2^f by the polynomial of degree 4 with the least relative error there (2.7e-6,
// fitted), n added to its exponent.  P is rounded to 2^-9 next, and the 32-bit sum
// of a row takes a quarter of its terms with that error: about a thousandth
// of what the rounding of P does to the output.  x below -126 (hidden scores are
// -inf) counts as -126, and 2^-126 is taken from all results.  That changes no
// weight above 2^-101 of its row's usual scale in 32 bits, and it leaves those at
// 1e-44, 0 as bf16, so that not even the largest finite value that nobody sees
// adds anything.
B200_DEV void exp2_pair(uint64_t x2, float& p0, float& p1) {
  const uint64_t magic = pair64(12582912.f, 12582912.f);
  float x0, x1;
  unpair64(x2, x0, x1);
  x2 = pair64(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t n2 = add2(x2, magic);
  const uint64_t f2 = add2(x2, add2(magic, n2 ^ 0x8000000080000000ull));
  uint64_t y = fma2(f2, pair64(0.009570100344717503f, 0.009570100344717503f), pair64(0.05591785907745361f, 0.05591785907745361f));
  y = fma2(y, f2, pair64(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, f2, pair64(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, f2, pair64(0.9999992847442627f, 0.9999992847442627f));
  float y0, y1, n0, n1;
  unpair64(y, y0, y1);
  unpair64(n2, n0, n1);
  y0 = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(n0) << 23));
  y1 = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(n1) << 23));
  unpair64(add2(pair64(y0, y1), pair64(-1.17549435e-38f, -1.17549435e-38f)), p0, p1);
}

// 32 scores to 2^(s scale - ref): 16 bf16 pairs in place (16 bits for the tensor
// core), the sums in 32 bits.  kPoly of 4 pairs go without the special-function
// unit, whose 16 results a cycle and SM would bound the kernel as the tensor core
// does: a key tile of both sides takes 3560 cycles with a quarter of them, 3760
// without.
constexpr int kPoly = 1;
B200_DEV void row_exp(uint32_t r[32], float scale_log2, float ref, uint64_t sums[2]) {
  const uint64_t scale2 = pair64(scale_log2, scale_log2), ref2 = pair64(-ref, -ref);
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint64_t x2 = fma2(pair64(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), scale2, ref2);
    float p0, p1;
    if (c % 4 >= 4 - kPoly) {
      exp2_pair(x2, p0, p1);
    } else {
      unpair64(x2, p0, p1);
      p0 = ex2(p0);
      p1 = ex2(p1);
    }
    sums[c & 1] = add2(sums[c & 1], pair64(p0, p1));
    r[c] = pack2(p0, p1);
  }
}

template <class P>
struct ItemsCfg {
  static constexpr int BOXES_QK = P::HDK / 64, BOXES_V = P::HDV / 64;
  static constexpr int TILE_QK = BOXES_QK * kBoxBytes, TILE_V = BOXES_V * kBoxBytes;
  static constexpr int K_STAGES = P::HDK > 128 ? 2 : P::HDK > 64 ? 3 : 4;
  static constexpr int V_STAGES = P::HDK > 128 ? 1 : P::HDK > 64 ? 2 : 4;
  static constexpr int K_AT = kSides * TILE_QK, V_AT = K_AT + K_STAGES * TILE_QK, BARS_AT = V_AT + V_STAGES * TILE_V;
  static constexpr int HIDDEN_AT = BARS_AT + 320;
  static constexpr int RING = 4 * V_STAGES;  // of the items' records
  static constexpr int SMEM = HIDDEN_AT + RING * (int)sizeof(Hidden) + 1024;
  static constexpr uint32_t IDESC_O = idesc_bf16_f32(128, P::HDV) | (1u << 16);  // B operand (V) MN-major
};

template <class P>
__global__ void __launch_bounds__(kItemThreads, 1)
    tc_items_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const P p, unsigned* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Cf = ItemsCfg<P>;
  constexpr int HDK = P::HDK, HDV = P::HDV, KS = Cf::K_STAGES, VS = Cf::V_STAGES;
  uint8_t* sK = smem + Cf::K_AT;
  uint8_t* sV = smem + Cf::V_AT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cf::BARS_AT);
  uint64_t* q_full = bars;           // [side] the item's Q landed
  uint64_t* q_empty = bars + 2;      // [side] the item's last scores are done: Q may be replaced
  uint64_t* s_full = bars + 4;       // [side] scores of a tile ready
  uint64_t* p_full = bars + 6;       // [side] P of a tile written (an arrival a softmax thread)
  uint64_t* pv_done = bars + 8;      // [side] P V of a tile done, and the list of zeroed keys behind it (2 arrivals)
  uint64_t* o_free = bars + 10;      // [side] the outputs are read out (an arrival a softmax thread)
  uint64_t* drain = bars + 12;       // [side] all MMAs issued, at the end
  uint64_t* turn = bars + 14;        // [side] it may issue
  uint64_t* k_full = bars + 16;      // [KS]
  uint64_t* k_empty = k_full + KS;   // [KS] (an arrival a side, as v_empty)
  uint64_t* v_full = k_empty + KS;   // [VS] landed
  uint64_t* v_ready = v_full + VS;   // [VS] and looked through
  uint64_t* v_empty = v_ready + VS;  // [VS]
  static_assert((16 + 2 * KS + 3 * VS) * 8 + 8 <= 320, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + VS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Hidden* hidden = reinterpret_cast<Hidden*>(smem + Cf::HIDDEN_AT);  // [item % Cf::RING]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // one value a warp
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSides; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 2);
      mbar_init(&o_free[s], 128);
      mbar_init(&drain[s], 1);
      mbar_init(&turn[s], 1);
    }
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    *abort_flag = 0;
    for (int i = 0; i < Cf::RING; ++i) hidden[i].any = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Inputs come from earlier kernels.  The wait stands before the TMEM
  // allocation, and the next kernel is let in after it: a kernel that holds
  // TMEM never waits for one that may be asking for it.
  pdl_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  typename P::Cursor cursor(p);
  typename P::Item it;

  if (warp == 0) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      bool ok = true;
      int g = 0, n[kSides] = {0, 0};  // tiles, and items of each side, so far
      int k_loads = 0, v_loads = 0;
      while (ok && !*abort_flag && cursor.next(it, err)) {
        for (int j = 0; ok && j < it.n; ++j, ++g) {
          const int ks = g % KS, vs = g % VS;
          if (g >= KS && !(ok = mbar_wait_idle(&k_empty[ks], (g / KS - 1) & 1, err))) break;
          P::load_k(p, it, j, sK + ks * Cf::TILE_QK, &tmK, &k_full[ks], err);
          ++k_loads;
          if (j == 0)
#pragma unroll
            for (int s = 0; s < kSides; ++s) {
              if (!ok || (s == 1 && !it.both)) break;
              if (n[s] > 0 && !(ok = mbar_wait_idle(&q_empty[s], (n[s] - 1) & 1, err))) break;
              P::load_q(p, it, s, smem + s * Cf::TILE_QK, &tmQ, &q_full[s]);
              ++n[s];
            }
          if (!ok) break;
          if (g >= VS && !(ok = mbar_wait_idle(&v_empty[vs], (g / VS - 1) & 1, err))) break;
          P::load_v(p, it, j, sV + vs * Cf::TILE_V, &tmV, &v_full[vs], err);
          ++v_loads;
        }
      }
      if (!ok) *abort_flag = 1;
      // whoever gives up before using a tile: no copy is in flight when the CTA ends
      for (int i = max(0, k_loads - KS); i < k_loads; ++i) mbar_wait_idle(&k_full[i % KS], (i / KS) & 1, err);
      for (int i = max(0, v_loads - VS); i < v_loads; ++i) mbar_wait_idle(&v_full[i % VS], (i / VS) & 1, err);
      for (int s = 0; s < kSides; ++s)
        if (n[s] > 0) mbar_wait_idle(&q_full[s], (n[s] - 1) & 1, err);
    }
    __syncwarp();
  } else if (warp == 1 || warp == kMma1Warp) {
    // ---------------- MMAs of a side ----------------
    // The sides take turns, a batch (P V, next scores) each: issued side by side,
    // both batches end together, and so both softmaxes begin together and leave
    // the tensor core without work.  A warp a side, so that one's waits and commits
    // pass while the other's batch runs.  A side's MMAs keep their order, which S
    // over the P before it needs; the sides touch different columns.
    const int s = warp == 1 ? 0 : 1;
    bool ok = true;
    int g = 0;           // the current item's first tile
    uint32_t n = 0;      // items of this side whose first scores were issued
    uint32_t t = 0;      // its tiles whose P V was issued
    uint32_t o = 0;      // its items whose P V began
    uint32_t o1 = 0;     // side 0: side 1's items before
    uint32_t turns = 0;  // of this side so far
    const uint32_t tS = tmem + kSideS + s * 128, tO = tmem + kSideO + s * 128;
    const uint64_t qd = smem_desc_k128(smem_u32(smem + s * Cf::TILE_QK));
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_idle(bar, parity, err)); };
    // (a thread that sleeps in a wait wakes 200 cycles later than one that polls)
    auto spin = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, err)); };
    // K of tile T and (of an item's first tile) Q have landed
    auto landed = [&](int T, bool first) {
      return (!first || wait(&q_full[s], n++ & 1)) && wait(&k_full[T % KS], (T / KS) & 1);
    };
    // S = Q K^T of tile T; `last` of its item
    auto scores = [&](int T, bool last) {
      const uint64_t kd = smem_desc_k128(smem_u32(sK + (T % KS) * Cf::TILE_QK));
#pragma unroll
      for (int k = 0; k < HDK / 16; ++k) {
        const uint64_t off = (uint64_t)(((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4);  // shared memory ends below 2^18
        umma_bf16_elect(tS, qd + off, kd + off, kIdescS, k > 0 ? 1u : 0u);
      }
      umma_commit_elect(&s_full[s]);
      umma_commit_elect(&k_empty[T % KS]);
      if (last) umma_commit_elect(&q_empty[s]);
    };
    // side 0 begins; then each waits until the other has issued its batch of a tile
    auto my_turn = [&] {
      const uint32_t k = turns++;
      return s == 0 ? k == 0 || wait(&turn[0], (k - 1) & 1) : wait(&turn[1], k & 1);
    };
    bool have = cursor.next(it, err);
    if (have) {
      const bool mine = s == 0 || it.both;
      ok = landed(0, mine);
      tc_fence_after();
      if (ok && mine) scores(0, it.n == 1);
      else if (ok) mbar_arrive_elect(&k_empty[0]);
    }
    while (ok && have && __all_sync(0xffffffffu, !*abort_flag)) {
      typename P::Item after;
      const bool more = cursor.next(after, err);
      const bool mine = s == 0 || it.both;
#pragma unroll 1
      for (int j = 0; ok && j < it.n; ++j) {
        const int T = g + j, vs = T % VS;
        const bool last = j + 1 == it.n;
        const bool next = !last || more;                          // scores of tile T + 1 are to come
        const bool next_mine = s == 0 || (last ? after.both : it.both);  // of this side
        // everything is waited for before the batch is issued, so that its products follow one another
        ok = (!next || landed(T + 1, last && next_mine)) && wait(&v_ready[vs], (T / VS) & 1);
        if (ok && mine && j == 0) {
          // all earlier items are stored (an item without side 1 waits for the last one that had it too)
          ok = (o == 0 || wait(&o_free[s], (o - 1) & 1)) && (it.both || o1 == 0 || wait(&o_free[1], (o1 - 1) & 1));
          ++o;
          o1 += it.both;
        }
        ok = ok && my_turn() && (!mine || spin(&p_full[s], t++ & 1));
        if (!ok) break;
        tc_fence_after();
        if (mine) {
          const uint64_t vd = smem_desc_mn128(smem_u32(sV + vs * Cf::TILE_V), kBoxBytes);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_bf16_ts_elect(tO, tS + k * 8, vd + (uint64_t)(k * 2048 >> 4), Cf::IDESC_O, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit_elect(&pv_done[s]);
        }
        if (next && next_mine) scores(T + 1, last ? after.n == 1 : j + 2 == it.n);
        mbar_arrive_elect(&turn[s ^ 1]);
        if (next && !next_mine) mbar_arrive_elect(&k_empty[(T + 1) % KS]);  // a tile that this side does not use
        if (mine) {
          mbar_arrive_elect(&pv_done[s]);
          umma_commit_elect(&v_empty[vs]);
        } else {
          mbar_arrive_elect(&v_empty[vs]);
        }
      }
      g += it.n;
      it = after;
      have = more;
    }
    // Whoever gave up, this warp or another whose flag ended the loop: every MMA issued completes before TMEM is freed.
    if (!ok) *abort_flag = 1;
    umma_commit_elect(&drain[s]);
    mbar_wait(&drain[s], 0, err);
    __syncwarp();
  } else if (warp == 2) {
    // ---------------- values looked through ----------------
    bool ok = true;
    int g = 0, n = 0;
#pragma unroll 1
    for (; ok && __all_sync(0xffffffffu, !*abort_flag) && cursor.next(it, err); ++n) {
      Hidden* hd = &hidden[n % Cf::RING];
      int edges = 0;
#pragma unroll 1
      for (int j = 0; j < it.n; ++j, ++g) {
        const int vs = g % VS;
        ok = __all_sync(0xffffffffu, mbar_wait_idle(&v_full[vs], (g / VS) & 1, err));
        if (!ok) break;
        // Records are cleared half a ring ahead of their use, once V of their item n has landed: it was loaded behind the
        // P V of item n - VS or a later one, and before an item's P V begins all earlier items have been stored (o_free).
        // So items up to n - VS - 1 are done with their records.  (Before this wait only V of item n - 1 has landed, and
        // with one stage the record, then of item n - 2, may still be read.)
        static_assert(VS + 1 <= Cf::RING / 2, "the record that item n clears belongs to item n - VS - 1 or an earlier one");
        if (j == 0 && lane == 0) hidden[(n + Cf::RING / 2) % Cf::RING].any = 0;
        const int key = P::key0(it, j);
        if (!P::whole(it, 0, key) || (it.both && !P::whole(it, 1, key))) {
          const int at = min(edges, kMaxEdgeTiles - 1);  // an item has six at most (row tiles in pairs: the window's start cuts three, the diagonal two, the sinks one)
          uint32_t any = 0;
#pragma unroll 1
          for (int w = 0; w < 4; ++w) {
            const uint32_t bad = clear_nonfinite<Cf::BOXES_V>(sV + vs * Cf::TILE_V + w * 32 * 128);
            if (lane == 0) hd->keys[at][w] = bad;
            any |= bad;
          }
          if (lane == 0) {
            hd->key0[at] = key;
            hd->count = at + 1;
            if (any) hd->any = 1;
          }
          ++edges;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ready[vs]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else {
    // ---------------- softmax ----------------
    // A thread a row, so no row's state leaves its thread.  (Two threads a row, eight
    // warps a side, took a tenth longer when both were timed, 310 us against 281 at
    // 8 x 2048: their exchange of maxima and the twice as many waits cost more than
    // the shorter rows gain.)
    const int s = (warp - 3) >> 2;           // side
    const int row = (warp & 3) * 32 + lane;  // TMEM lanes that this warp may access: 32 (warp % 4) ..
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + kSideS + s * 128, tO = tmem + lanes + kSideO + s * 128;
    const float scale_log2 = p.scale_log2;
    bool ok = true;
    int t = 0, n = 0;  // tiles of this side, and items, so far
#pragma unroll 1
    for (; ok && cursor.next(it, err); ++n) {
      if (s == 1 && !it.both) continue;
      float mref = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < it.n; ++j, ++t) {
        // warp-uniform: TMEM's accesses are
        ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait_idle(&s_full[s], t & 1, err));
        if (!ok) break;
        tc_fence_after();
        const int key = P::key0(it, j);
        const bool edge = !P::whole(it, s, key);
        uint32_t ra[32], rb[32];
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        // The scores are read from TMEM twice, 32 columns at a time with the next 32 on
        // their way: once for the maximum, once for the exponentials.  Held from the
        // one to the other, they would make the code of a tile several times longer
        // than the instruction cache likes.
        uint32_t unseen = 0;  // edge tiles: bit c: no row of this warp sees columns 32 c ..
        if (!edge) {
          tmem_ld_32x32b_x32(tS, ra);
#pragma unroll 1
          for (int c = 0; c < 4; c += 2) {
            tmem_ld_wait();
            tmem_ld_32x32b_x32(tS + (c + 1) * 32, rb);
            row_max(ra, m4);
            tmem_ld_wait();
            tmem_ld_32x32b_x32(tS + ((c + 2) & 3) * 32, ra);  // at the end the first again
            row_max(rb, m4);
          }
        } else {
          // hidden scores become -inf where they lie; columns that the warp does not see are left out
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const uint32_t mask = P::visible(it, s, row, key + c * 32);
            if (__all_sync(0xffffffffu, mask == 0)) {
              unseen |= 1u << c;
              continue;
            }
            tmem_ld_32x32b_x32(tS + c * 32, ra);
            tmem_ld_wait();
            if (!__all_sync(0xffffffffu, mask == 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((mask >> i) & 1u)) ra[i] = __float_as_uint(-INFINITY);
              tmem_st_32x32b_x32(tS + c * 32, ra);
            }
            row_max(ra, m4);
          }
          tmem_st_wait();
        }
        float mx = fmax3_nan(fmax3_nan(m4[0], m4[1], m4[2]), m4[3], -INFINITY);
        if (!(mx < INFINITY)) l = NAN;  // a visible score is NaN or +inf (inf / inf): so is the row
        mx *= scale_log2;       // scale > 0
        float alpha = 1.f;
        if (mx > mref + kRescaleLog2 || (mref == -INFINITY && mx > -INFINITY)) {
          if (mref != -INFINITY) alpha = ex2(mref - mx);
          l *= alpha;  // 0 so far where there was no maximum
          mref = mx;
        }
        const float ref = mref == -INFINITY ? 0.f : mref;
        uint64_t sums[2] = {0, 0};
        // P of 32 scores takes 16 columns, over scores that have been read
        if (!edge) {
#pragma unroll 1
          for (int c = 0; c < 4; c += 2) {
            tmem_ld_wait();
            tmem_ld_32x32b_x32(tS + (c + 1) * 32, rb);
            row_exp(ra, scale_log2, ref, sums);
            tmem_st_32x32b_x16(tS + c * 16, ra);
            tmem_ld_wait();
            if (c == 0) tmem_ld_32x32b_x32(tS + 64, ra);
            row_exp(rb, scale_log2, ref, sums);
            tmem_st_32x32b_x16(tS + c * 16 + 16, rb);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            if ((unseen >> c) & 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) ra[i] = 0;
            } else {
              tmem_ld_32x32b_x32(tS + c * 32, ra);
              tmem_ld_wait();
              row_exp(ra, scale_log2, ref, sums);
            }
            tmem_st_32x32b_x16(tS + c * 16, ra);
          }
        }
        float l0, l1;
        unpair64(add2(sums[0], sums[1]), l0, l1);
        l += l0 + l1;
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // O holds the item's tiles before j once the last of them is done
          ok = __all_sync(0xffffffffu, mbar_wait_idle(&pv_done[s], (t - 1) & 1, err));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HDV / 32; ++c) {
            tmem_ld_32x32b_x32(tO + c * 32, ra);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) ra[i] = __float_as_uint(__uint_as_float(ra[i]) * alpha);
            tmem_st_32x32b_x32(tO + c * 32, ra);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[s]);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait_idle(&pv_done[s], (t - 1) & 1, err));
      if (!ok) break;
      const volatile Hidden* hd = &hidden[n % Cf::RING];
#pragma unroll 1
      for (int i = 0; i < (hd->any ? hd->count : 0); ++i)  // zeroed keys that this row sees
#pragma unroll 1
        for (int w = 0; w < 4; ++w)
          if (P::visible(it, s, row, hd->key0[i] + 32 * w) & hd->keys[i][w]) l = NAN;
      tc_fence_after();
      P::store(p, it, s, row, mref, l, tO);
      tc_fence_before();
      mbar_arrive(&o_free[s]);
    }
    if (!ok) *abort_flag = 1;
    tmem_ld_wait();  // nothing of a tile that was given up is on its way when TMEM is freed
    tmem_st_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <class P>
int launch_items(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const P& p, int grid,
                 cudaStream_t st) {
  auto k = tc_items_kernel<P>;
  constexpr int smem = ItemsCfg<P>::SMEM;
  static_assert(smem <= 227 * 1024, "shared memory");
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERROR_UNSUPPORTED;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return B200_ERROR_UNSUPPORTED;
    done[dev] = true;
  }
  launch_kernel(k, dim3((unsigned)grid), kItemThreads, smem, st, mq, mk, mv, p, b200::error_word(dev));
  B200_CHECK_LAUNCH();
  return B200_OK;
}

inline int sm_count() {
  static int n[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] > 0 ? n[dev] : 148;
}

}  // namespace

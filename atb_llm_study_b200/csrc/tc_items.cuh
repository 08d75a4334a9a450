// Attention of query tiles over lists of key tiles on the tcgen05 tensor cores:
// the kernel of sliding-window prompts and of shared prefixes.
//
//   out = sum_j p_j v_j / sum_j p_j, p_j = 2^(q.k_j scale log2(e) - m)
//
// One item is 128 query rows and a list of 128-key tiles; a persistent CTA per
// SM walks its items.  The roles are those of the whole-prompt kernel
// (flash_tc.cu): a TMA warp, a thread that issues the scores S = Q K^T into
// three TMEM buffers, eight softmax warps with two threads a row that write P
// over their scores, and a warp that issues O += P V.  What an item's rows and
// keys are, which pairs see each other and where the output goes is the
// problem's (P below).
//
// Values that nobody sees must not reach anybody: P is 0 there, but 0 x NaN is
// not.  So the P.V warp looks through the value rows of every tile that is not
// visible as a whole (the edges: a prompt's end, its diagonal, the ends of the
// window and the sinks, a cache block's rest) and zeroes those with a NaN or an
// infinity.  A row that does see such a key gets NaN: the item's list of zeroed
// keys is looked through when its rows are stored.  The search takes one warp
// 64 loads and ballots a tile while the tile's scores are computed.
//
// P provides: HDK, HDV; Item with `int n` (key tiles, > 0); Cursor(p) with
// bool next(Item&, err); load_q / load_k / load_v(p, item, [tile,] smem, map, bar, err):
// arrive on bar expecting bytes, copy; int key0(item, tile): its first key;
// bool whole(item, key, keys): every row sees all of [key, key + keys);
// bool sees(item, row, key); store(p, item, row, half, m, l, tO).
#pragma once

#include "tc_attention.cuh"

namespace {

struct Hidden {  // zeroed value rows of one item's edge tiles
  int count;
  int key0[6];
  uint32_t keys[6][4];
};
constexpr int kMaxEdgeTiles = 6;

// Zeroes the rows of a V tile [128 keys] that hold a NaN or an infinity; keys' bits of those in `bad`.  One warp.
template <int BOXES>
B200_DEV bool clear_nonfinite(uint8_t* sV, uint32_t bad[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad[i] = 0;
  // an instruction covers 4 rows, 8 lanes of 16 bytes a row; rows are 128 contiguous bytes whatever the swizzle
#pragma unroll 1
  for (int w = 0; w < 4; ++w) {
    uint32_t found = 0;
#pragma unroll
    for (int x = 0; x < BOXES; ++x)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(sV + x * kBoxBytes + (w * 32 + i * 4) * 128 + lane * 16);
        // exponent bits all ones: 0x7f80 + 0x80 carries into bit 15
        uint32_t t = (v.x & 0x7f807f80u) + 0x00800080u;
        t |= (v.y & 0x7f807f80u) + 0x00800080u;
        t |= (v.z & 0x7f807f80u) + 0x00800080u;
        t |= (v.w & 0x7f807f80u) + 0x00800080u;
        const uint32_t lanes = __ballot_sync(0xffffffffu, (t & 0x80008000u) != 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (lanes & (0xffu << (8 * r))) found |= 1u << (i * 4 + r);
      }
    bad[w] = found;
    if (found)
#pragma unroll 1
      for (int r = 0; r < 32; ++r)
        if ((found >> r) & 1u)
          for (int c = lane; c < BOXES * 8; c += 32)
            *reinterpret_cast<uint4*>(sV + (c >> 3) * kBoxBytes + (w * 32 + r) * 128 + (c & 7) * 16) =
                make_uint4(0, 0, 0, 0);
  }
  const bool any = (bad[0] | bad[1] | bad[2] | bad[3]) != 0;
  if (any) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor core reads the tile
  __syncwarp();
  return any;
}

template <class P>
struct ItemsCfg {
  using Tc = TcCfg<P::HDK, P::HDV>;
  static constexpr int HIDDEN = Tc::SMEM - 1024;  // behind tiles, exchange and barriers
  static constexpr int SMEM = Tc::SMEM + 2 * (int)sizeof(Hidden);
};

template <class P>
__global__ void __launch_bounds__(kThreads, 1)
    tc_items_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const P p, unsigned* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Cf = TcCfg<P::HDK, P::HDV>;
  constexpr int HDK = P::HDK, HDV = P::HDV;
  constexpr int kTileBytes = Cf::TILE_QK, kVBytes = Cf::TILE_V, VS = Cf::V_STAGES;
  uint8_t* sQ = smem;
  uint8_t* sK = smem + kTileBytes;
  uint8_t* sV = smem + 3 * kTileBytes;
  float* sMx = reinterpret_cast<float*>(sV + VS * kVBytes);  // [tile parity][half][row]
  float* sL = sMx + 4 * 128;                                  // [half][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sL + 2 * 128);
  uint64_t* q_full = bars;        // Q of the current item landed
  uint64_t* q_empty = bars + 1;   // the item's last scores done: Q may be replaced
  uint64_t* k_full = bars + 2;    // [2]
  uint64_t* k_empty = bars + 4;   // [2]
  uint64_t* v_full = bars + 6;    // [2]
  uint64_t* v_empty = bars + 8;   // [2]
  uint64_t* s_full = bars + 10;   // [3] scores of the tile in buffer i ready
  uint64_t* p_full = bars + 13;   // [3] P of the tile in buffer i written (256 arrivals)
  uint64_t* pv_done = bars + 16;  // [3] P.V of the tile whose P sits in buffer i done
  uint64_t* o_free = bars + 19;   // the output accumulator read out (256 arrivals)
  uint64_t* drain = bars + 20;    // [2] MMA issuers' teardown after an abort
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Hidden* hidden = reinterpret_cast<Hidden*>(smem + ItemsCfg<P>::HIDDEN);  // [item parity]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kSBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 256);
      mbar_init(&pv_done[i], 2);  // the products, and the thread whose list of zeroed keys goes with them
    }
    mbar_init(o_free, 256);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
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
  const uint32_t tmem = *tmem_slot;
  typename P::Cursor cursor(p);
  typename P::Item it;

  if (warp == 0) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      bool ok = true;
      int g = 0, n = 0;  // tiles and items so far
      for (; ok && !*abort_flag && cursor.next(it, err); ++n) {
        for (int j = 0; j < it.n; ++j, ++g) {
          const int st = g & 1, vst = g % VS;
          if (g >= 2 && !(ok = mbar_wait_idle(&k_empty[st], ((g >> 1) & 1) ^ 1, err))) break;
          P::load_k(p, it, j, sK + st * kTileBytes, &tmK, &k_full[st], err);
          if (j == 0) {
            if (n > 0 && !(ok = mbar_wait_idle(q_empty, (n - 1) & 1, err))) break;
            P::load_q(p, it, sQ, &tmQ, q_full);
          }
          if (g >= VS && !(ok = mbar_wait_idle(&v_empty[vst], ((g / VS) & 1) ^ 1, err))) break;
          P::load_v(p, it, j, sV + vst * kVBytes, &tmV, &v_full[vst], err);
        }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- scores ----------------
    if (lane == 0) {
      bool ok = true;
      int g = 0, n = 0;
      for (; ok && !*abort_flag && cursor.next(it, err); ++n) {
        if (!(ok = mbar_wait_idle(q_full, n & 1, err))) break;
        for (int j = 0; j < it.n; ++j, ++g) {
          const int b = g % kSBufs, u = g / kSBufs;
          ok = mbar_wait_idle(&k_full[g & 1], (g >> 1) & 1, err) &&
               (g < kSBufs || mbar_wait_idle(&pv_done[b], (u - 1) & 1, err));
          if (!ok) break;
          tc_fence_after();
          const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK + (g & 1) * kTileBytes);
#pragma unroll
          for (int ks = 0; ks < HDK / 16; ++ks) {
            const uint32_t off = (ks >> 2) * kBoxBytes + (ks & 3) * 32;
            umma_bf16(tmem + b * 128, smem_desc_k128(q0 + off), smem_desc_k128(k0 + off), kIdescS, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[b]);
          umma_commit(&k_empty[g & 1]);
          if (j + 1 == it.n) umma_commit(q_empty);
        }
      }
      if (!ok) {
        *abort_flag = 1;
        umma_commit(&drain[0]);  // every MMA issued by this thread completes before TMEM is freed
        mbar_wait(&drain[0], 0, err);
      }
    }
    __syncwarp();
  } else if (warp == kPvWarp) {
    // ---------------- P.V (a whole warp: it also clears edge tiles) ----------------
    bool ok = true;
    int g = 0, n = 0;
    for (; ok && !*abort_flag && cursor.next(it, err); ++n) {
      Hidden* hd = &hidden[n & 1];  // last read before item n - 2 let the accumulator go: see the wait on o_free
      if (lane == 0) hd->count = 0;
      __syncwarp();
      for (int j = 0; j < it.n; ++j, ++g) {
        const int b = g % kSBufs, vst = g % VS;
        ok = mbar_wait_idle(&v_full[vst], (g / VS) & 1, err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (!P::whole(it, P::key0(it, j), kTile)) {
          uint32_t bad[4];
          if (clear_nonfinite<Cf::BOXES_V>(sV + vst * kVBytes, bad) && lane == 0 && hd->count < kMaxEdgeTiles) {
            const int at = hd->count;
            hd->key0[at] = P::key0(it, j);
            for (int i = 0; i < 4; ++i) hd->keys[at][i] = bad[i];
            hd->count = at + 1;
          }
          __syncwarp();
        }
        ok = mbar_wait_idle(&p_full[b], (g / kSBufs) & 1, err) &&
             (j > 0 || n == 0 || mbar_wait_idle(o_free, (n - 1) & 1, err));
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          tc_fence_after();
          const uint32_t pa = tmem + b * 128, v0 = smem_u32(sV + vst * kVBytes);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            umma_bf16_ts(tmem + kOCol, pa + (ks >> 2) * 64 + (ks & 3) * 8, smem_desc_mn128(v0 + ks * 2048, kBoxBytes),
                         Cf::IDESC_O, (j > 0 || ks > 0) ? 1u : 0u);
          umma_commit(&pv_done[b]);
          umma_commit(&v_empty[vst]);
          mbar_arrive(&pv_done[b]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) {
        umma_commit(&drain[1]);
        mbar_wait(&drain[1], 0, err);
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax (warps 2..9: two threads per query row) ----------------
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    const int half = (warp - 2) >> 2;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int pair_bar = 1 + quarter;  // named barrier of warps (quarter + 2, quarter + 6)
    const float scale_log2 = p.scale_log2;
    bool ok = true;
    int g = 0, n = 0;
    for (; ok && cursor.next(it, err); ++n) {
      const uint32_t tO = tmem + lanes + kOCol + half * (HDV / 2);
      float mref = -INFINITY, l = 0.f;
      for (int j = 0; j < it.n; ++j, ++g) {
        const int st = g % kSBufs;
        // the same outcome for both warps of the pair (they meet at named barriers)
        const bool got = __all_sync(0xffffffffu, ok && !*abort_flag && mbar_wait_idle(&s_full[st], (g / kSBufs) & 1, err));
        if (pair_or(pair_bar, !got)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[64];
        tmem_ld_32x32b_x32(tmem + lanes + st * 128 + half * 64, sr);
        tmem_ld_32x32b_x32(tmem + lanes + st * 128 + half * 64 + 32, sr + 32);
        tmem_ld_wait();
        const int key = P::key0(it, j) + half * 64;  // first key of this thread's columns
        if (!P::whole(it, key, 64)) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (!P::sees(it, row, key + c)) sr[c] = __float_as_uint(-INFINITY);
        }
        // raw-score max of this half (scale > 0): eight independent chains of three-input maxima
        float m8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmax3(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1]), -INFINITY);
#pragma unroll
        for (int c = 8; c < 32; ++c)
          m8[c & 7] = fmax3(m8[c & 7], __uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1]));
        float mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
        sMx[((g & 1) * 2 + half) * 128 + row] = mx;
        named_bar_sync(pair_bar, 64);
        mx = fmaxf(mx, sMx[((g & 1) * 2 + (half ^ 1)) * 128 + row]);
        mx *= scale_log2;
        // the running max moves only when it grows by more than 2^kRescaleLog2
        float alpha = 1.f;
        bool rescale = false;
        if (mx > mref + kRescaleLog2 || (mref == -INFINITY && mx > -INFINITY)) {
          rescale = mref != -INFINITY;
          alpha = rescale ? ex2(mref - mx) : 0.f;
          l *= alpha;
          mref = mx;
        }
        const float ref = mref == -INFINITY ? 0.f : mref;
        float r8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r8[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float p0 = ex2(fmaf(__uint_as_float(sr[2 * c]), scale_log2, -ref));
          const float p1 = ex2(fmaf(__uint_as_float(sr[2 * c + 1]), scale_log2, -ref));
          r8[c & 7] += p0 + p1;
          sr[c] = pack2(p0, p1);
        }
        l += ((r8[0] + r8[1]) + (r8[2] + r8[3])) + ((r8[4] + r8[5]) + (r8[6] + r8[7]));
        if (j > 0 && __any_sync(0xffffffffu, rescale)) {
          // a failed wait is acted on at the next tile's pair vote (no exit between pair barriers)
          if (!__all_sync(0xffffffffu, mbar_wait_idle(&pv_done[(g - 1) % kSBufs], ((g - 1) / kSBufs) & 1, err)))
            ok = false;
          tc_fence_after();
          if (ok) {
#pragma unroll 1
            for (int c = 0; c < HDV / 64; ++c) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(tO + c * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * (rescale ? alpha : 1.f));
              tmem_st_32x32b_x32(tO + c * 32, r);
            }
            tmem_st_wait();
          }
        }
        tmem_st_32x32b_x32(tmem + lanes + st * 128 + half * 64, sr);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[st]);
      }
      const bool done = __all_sync(0xffffffffu, ok && !*abort_flag &&
                                                    mbar_wait_idle(&pv_done[(g - 1) % kSBufs], ((g - 1) / kSBufs) & 1, err));
      if (pair_or(pair_bar, !done)) {
        ok = false;
        break;
      }
      sL[half * 128 + row] = l;
      named_bar_sync(pair_bar, 64);
      l += sL[(half ^ 1) * 128 + row];
      named_bar_sync(pair_bar, 64);  // sL is rewritten at the next item's end
      const volatile Hidden* hd = &hidden[n & 1];
      for (int i = 0; i < hd->count; ++i)  // zeroed keys that this row sees
        for (int c = 0; c < 128; ++c)
          if (((hd->keys[i][c >> 5] >> (c & 31)) & 1u) && P::sees(it, row, hd->key0[i] + c)) l = NAN;
      tc_fence_after();
      P::store(p, it, row, half, mref, l, tO);
      tc_fence_before();
      mbar_arrive(o_free);
    }
    if (!ok) *abort_flag = 1;
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
  launch_kernel(k, dim3((unsigned)grid), kThreads, smem, st, mq, mk, mv, p, b200::error_word(dev));
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

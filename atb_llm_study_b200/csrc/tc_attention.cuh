// Shared pieces of the tcgen05 attention kernels: the warp roles' constants, shared-memory sizes, descriptors, TMEM
// stores, barriers of warp pairs and the tensor maps of packed operands.
#pragma once

#include <math.h>

#include "common.cuh"
#include "tensor_map.h"

namespace {

using namespace b200;

constexpr int kThreads = 352;  // warps: 0 TMA, 1 score MMAs, 2-9 softmax, 10 P.V MMAs
constexpr int kPvWarp = 10;
constexpr int kTile = 128;                    // query rows per CTA = keys per tile
constexpr int kBoxBytes = kTile * 128;        // 128 rows x 64 bf16 (one 128-byte swizzle span)
constexpr int kXBytes = (4 + 2) * 128 * 4;    // row-half exchange: maxima [2 tiles][2 halves], sums [2 halves]
// query/key head width HDK (64, 128 or 192) and value width HDV (64 or 128):
// Q and K tiles are HDK / 64 boxes of 128 rows, V tiles HDV / 64 boxes
template <int HDK, int HDV>
struct TcCfg {
  static constexpr int BOXES_QK = HDK / 64, BOXES_V = HDV / 64;
  static constexpr int TILE_QK = BOXES_QK * kBoxBytes, TILE_V = BOXES_V * kBoxBytes;
  static constexpr int V_STAGES = HDK > 128 ? 1 : 2;
  // Q, K x2, V x V_STAGES, P + alignment + barriers
  static constexpr int SMEM = 3 * TILE_QK + V_STAGES * TILE_V + kXBytes + 1024 + 256;
  static constexpr uint32_t IDESC_O = idesc_bf16_f32(128, HDV) | (1u << 16);  // B operand (V) MN-major
};
constexpr uint32_t kTmemCols = 512;           // score / P buffers at [0,128) [128,256) [256,384), O at [384,512)
constexpr int kSBufs = 3;
constexpr uint32_t kOCol = 384;
constexpr float kRescaleLog2 = 8.f;           // move the running max only when it grows by > 2^8
constexpr uint32_t kIdescS = idesc_bf16_f32(128, 128);

// MN-major operand, 128-byte swizzle: 64-element rows of the MN dimension,
// 8-row groups of the K dimension 1024 bytes apart (SBO), the next 64
// MN elements `lbo` bytes away (LBO).
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t r[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x on the special-function unit (PTX ex2.approx, relative error ~2^-22)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D[tmem] (+)= A[tmem] * B[smem desc]^T, kind::f16: A (M x K, bf16 pairs per
// 32-bit column, row m in lane m) read from tensor memory.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// ---- The same issued by one elected lane (always the same) of a converged warp
// whose values agree.  Their operands are then known to be one for the whole warp
// and stay in the uniform registers that the instruction reads: 64 cycles an MMA
// of 128 x 128 x 16, the tensor core's own pace.  In code that a single thread
// has branched to, each operand is moved there instruction by instruction, and an
// MMA takes 150 cycles to issue (measured, batches of 8). ----
__device__ __forceinline__ void umma_bf16_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_ts_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                   uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b64 st;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// max(a, b, c) in one instruction (three-input max.f32 of sm_100)
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Named barrier `id` over `n` threads.
__device__ __forceinline__ void named_bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
// Named barrier `id` over 64 threads returning the OR of `v` over them.
__device__ __forceinline__ bool pair_or(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)v)
      : "memory");
  return r != 0;
}

// Row-major bf16 [rows, cols] with row stride ld (elements); box = 128 rows x
// 64 columns, 128-byte swizzle; rows past `rows` read as zeros.
inline bool make_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int64_t ld) {
  return encode_tiled_2d(m, ptr, cols, rows, ld * 2, 64, kTile);
}

// [rows][heads][hd] view of a row-major bf16 matrix (row stride ld, head
// stride hs, elements) for heads narrower than 64: box = 64 x 1 head x 128
// rows, the 64 - hd columns past each head and rows past `rows` read as zeros.
inline bool make_map_heads(CUtensorMap* m, const void* ptr, int64_t rows, int64_t heads, int64_t hd, int64_t hs,
                           int64_t ld) {
  return encode_tiled_3d(m, ptr, hd, heads, rows, hs * 2, ld * 2, 64, 1, kTile);
}

}  // namespace

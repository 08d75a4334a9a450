// Rows of bf16 values to 8-bit integers with one scale a row: the operand of
// the 8-bit products, made from activations (per token) and from weights (per
// output channel) alike.  Reads 2 bytes and writes 1 byte a value, and is bound
// by that: 16384 x 12288 in 86 us (604 MB, 7.0 TB/s), 49152 rows of 2048 gathered
// from 8192 in 31 us (134 MB at DRAM, and 201 MB read out of L2), 49152 x 1408 in 33 us (207 MB, 6.3 TB/s); one row, or 64 of
// 4096, in 3.2 us, the length of a launch.  (A rounding and a conversion
// instruction a value, both on the slow conversion pipe, took 137 us for the
// first; one FMA does both, see quant.cuh.)
#include "quant.cuh"

using namespace b200;

namespace {

struct QuantParams {
  const __nv_bfloat16* x;
  int64_t ldx;
  const int32_t* src;    // row of x for each output row (NULL: the same row)
  int64_t src_rows;
  const int32_t* count;  // output rows at or above *count are left alone (NULL: none are)
  int8_t* q;
  int64_t ldq;
  float* scale;
  int64_t rows, dim;
  unsigned* err;
};

// The x row of output row `row`, or NULL when there is nothing to write.
__device__ __forceinline__ const __nv_bfloat16* source_row(const QuantParams& p, int64_t row, bool leader) {
  if (p.count && row >= *p.count) return nullptr;
  int64_t sr = row;
  if (p.src) {
    sr = p.src[row];
    if (sr < 0 || sr >= p.src_rows) {
      if (leader) raise_error(p.err, DEV_ERR_BAD_INDEX);
      return nullptr;
    }
  }
  return p.x + sr * p.ldx;
}

// W warps per row (1: the rows of a CTA's four warps are apart and nothing is
// exchanged through shared memory).  The row stays in registers between its
// maximum and the write; a thread owns CH chunks of 16 values (32 bytes read,
// 16 written).
template <int W, int CH>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) quant_rows_kernel(const QuantParams p) {
  __shared__ uint32_t red[W];
  pdl_trigger();
  pdl_wait();
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int t = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  if (row >= p.rows) return;
  const __nv_bfloat16* xr = source_row(p, row, t == 0);
  if (!xr) return;
  uint4 v[CH][2];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = ((int64_t)c * (W * 32) + t) * 16;
    if (i < p.dim) {
      v[c][0] = *reinterpret_cast<const uint4*>(xr + i);
      v[c][1] = *reinterpret_cast<const uint4*>(xr + i + 8);
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = ((int64_t)c * (W * 32) + t) * 16;
    if (i < p.dim) m = amax_pairs(amax_pairs(m, v[c][0]), v[c][1]);
  }
  const RowQuant r = row_quant(W == 1 ? warp_amax(m) : block_amax<W * 32>(m, red));
  if (t == 0) p.scale[row] = r.scale;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = ((int64_t)c * (W * 32) + t) * 16;
    if (i < p.dim) {
      const uint2 a = quant8(v[c][0], r), b = quant8(v[c][1], r);
      *reinterpret_cast<uint4*>(p.q + row * p.ldq + i) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

// Rows too long for registers: the second pass reads the row again (from L2).
constexpr int kLongThreads = 512;
__global__ void __launch_bounds__(kLongThreads) quant_long_rows_kernel(const QuantParams p) {
  __shared__ uint32_t red[kLongThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const __nv_bfloat16* xr = source_row(p, row, threadIdx.x == 0);
  if (!xr) return;
  uint32_t m = 0;
  for (int64_t i = threadIdx.x * 8; i < p.dim; i += kLongThreads * 8)
    m = amax_pairs(m, *reinterpret_cast<const uint4*>(xr + i));
  const RowQuant r = row_quant(block_amax<kLongThreads>(m, red));
  if (threadIdx.x == 0) p.scale[row] = r.scale;
  for (int64_t i = threadIdx.x * 16; i < p.dim; i += kLongThreads * 16) {
    const uint2 a = quant8(*reinterpret_cast<const uint4*>(xr + i), r);
    const uint2 b = quant8(*reinterpret_cast<const uint4*>(xr + i + 8), r);
    *reinterpret_cast<uint4*>(p.q + row * p.ldq + i) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" int b200_quant_rows_int8(const void* x, int64_t ldx, int64_t src_rows, const int32_t* row_src,
                                    const int32_t* row_count, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                                    int64_t dim, b200_stream_t stream) {
  if (!x || !q || !scale || rows < 0 || src_rows < 0 || dim <= 0 || dim % 16 || ldx < dim || ldx % 8 || ldq < dim ||
      ldq % 16)
    return B200_ERROR_INVALID_PARAM;
  if (!row_src && src_rows < rows) return B200_ERROR_INVALID_PARAM;
  if (!aligned16(x) || !aligned16(q) || ((uintptr_t)scale & 3u) || ((uintptr_t)row_src & 3u) ||
      ((uintptr_t)row_count & 3u))
    return B200_ERROR_INVALID_PARAM;
  if (rows > INT32_MAX) return B200_ERROR_UNSUPPORTED;
  if (rows == 0) return B200_OK;
  int dev = 0;
  cudaGetDevice(&dev);
  const QuantParams p{static_cast<const __nv_bfloat16*>(x), ldx, row_src, src_rows, row_count, q, ldq, scale, rows, dim,
                      b200::error_word(dev)};
  const dim3 g((unsigned)rows), g4((unsigned)((rows + 3) / 4));
  // Many short rows: a warp each, four chunks at most (49152 x 1408 33 us, with a
  // CTA of four warps a row 66).  Otherwise the row's CTA is sized for two to four
  // chunks a thread, so that few rows are loaded by many threads at once.
  const bool many = rows >= 4096;
  if (many && dim <= 512) launch_kernel(quant_rows_kernel<1, 1>, g4, 128, 0, stream, p);
  else if (many && dim <= 1024) launch_kernel(quant_rows_kernel<1, 2>, g4, 128, 0, stream, p);
  else if (many && dim <= 2048) launch_kernel(quant_rows_kernel<1, 4>, g4, 128, 0, stream, p);
  else if (dim <= 2048) launch_kernel(quant_rows_kernel<4, 1>, g, 128, 0, stream, p);
  else if (dim <= 4096) launch_kernel(quant_rows_kernel<4, 2>, g, 128, 0, stream, p);
  else if (dim <= 8192) launch_kernel(quant_rows_kernel<8, 2>, g, 256, 0, stream, p);
  else if (dim <= 16384) launch_kernel(quant_rows_kernel<8, 4>, g, 256, 0, stream, p);
  else launch_kernel(quant_long_rows_kernel, g, kLongThreads, 0, stream, p);
  B200_CHECK_LAUNCH();
  return B200_OK;
}

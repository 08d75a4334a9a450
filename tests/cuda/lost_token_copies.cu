// paged_window_kernel with tensor maps whose boxes may be shorter than the tiles that the kernel announces to its
// barriers: the rest of each copy never comes, the waits behind it run out, and the kernel has to end by itself with its
// error word set.
#include "paged_window.cu"

namespace b200 {
bool pdl_enabled() { return false; }
unsigned* error_word(int) { return nullptr; }
}  // namespace b200

extern "C" __attribute__((visibility("default"))) int lost_token_copy(const void* q, const void* k, const void* v,
                                                                      const int32_t* tables, int width,
                                                                      const int32_t* context, int batch, int nq, int nkv,
                                                                      int block_size, int num_blocks, int window, void* out,
                                                                      unsigned ctas, int box_rows, unsigned* err,
                                                                      cudaStream_t stream) {
  constexpr int HD = 64;
  Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = p.out_stride = nq * HD;
  p.tables = tables;
  p.width = width;
  p.context = context;
  p.nq = nq;
  p.nkv = nkv;
  p.group = nq / nkv;
  p.head_tiles = (p.group + kRows - 1) / kRows;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.scale_log2 = 0.125f * kLog2e;
  p.window = window;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.err = err;
  CUtensorMap tk, tv;
  const int64_t rows = (int64_t)num_blocks * nkv * block_size;
  if (!encode_tiled_2d(&tk, k, HD, rows, HD * 2, 64, kTile) || !encode_tiled_2d(&tv, v, HD, rows, HD * 2, 64, box_rows))
    return -1;
  auto kernel = paged_window_kernel<HD>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM) != cudaSuccess) return -2;
  return (int)launch_clusters(kernel, ctas, dim3(batch * nkv * p.head_tiles * ctas), kThreads, Cfg<HD>::SMEM, stream, tk,
                              tv, p);
}

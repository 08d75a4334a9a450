// tc_items_kernel over plain attention, with one TMA copy that is announced to its barrier and never issued: the waits
// behind it run out, and the kernel has to end by itself with its error word set.
#include "tc_items.cuh"

namespace b200 {
bool pdl_enabled() { return false; }
unsigned* error_word(int) { return nullptr; }
}  // namespace b200

namespace {

enum Operand { kNone, kQ, kK, kV };

struct Plain {
  static constexpr int HDK = 64, HDV = 64;
  using Cf = ItemsCfg<Plain>;
  __nv_bfloat16* out;  // [items * 256][64]
  int items, keys;
  float scale_log2;
  int lost, lost_item, lost_tile;

  struct Item {
    int n, index, keys;
    bool both;
  };
  struct Cursor {
    const Plain& p;
    int w;
    B200_DEV explicit Cursor(const Plain& q) : p(q), w(blockIdx.x) {}
    B200_DEV bool next(Item& it, unsigned*) {
      if (w >= p.items) return false;
      it = Item{(p.keys + kTile - 1) / kTile, w, p.keys, true};
      w += gridDim.x;
      return true;
    }
  };
  B200_DEV static int key0(const Item&, int j) { return j * kTile; }
  B200_DEV static bool whole(const Item& it, int, int key) { return key + kTile <= it.keys; }
  B200_DEV static uint32_t visible(const Item& it, int, int, int key) { return bit_range(0, it.keys - key); }
  B200_DEV static void copy(bool lost, uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row) {
    mbar_arrive_expect_tx(bar, kBoxBytes);
    if (!lost) tma_load_2d(dst, map, bar, 0, row);
  }
  B200_DEV static void load_q(const Plain& p, const Item& it, int s, uint8_t* dst, const CUtensorMap* map, uint64_t* bar) {
    copy(p.lost == kQ && it.index == p.lost_item && s == p.lost_tile, dst, map, bar, (2 * it.index + s) * kTile);
  }
  B200_DEV static void load_k(const Plain& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                              unsigned*) {
    copy(p.lost == kK && it.index == p.lost_item && j == p.lost_tile, dst, map, bar, j * kTile);
  }
  B200_DEV static void load_v(const Plain& p, const Item& it, int j, uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                              unsigned*) {
    copy(p.lost == kV && it.index == p.lost_item && j == p.lost_tile, dst, map, bar, j * kTile);
  }
  B200_DEV static void store(const Plain& p, const Item& it, int s, int row, float, float l, uint32_t tO) {
    __nv_bfloat16* o = p.out + ((int64_t)(2 * it.index + s) * kTile + row) * HDV;
    for (int c = 0; c < HDV / 32; ++c) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tO + c * 32, r);
      tmem_ld_wait();
      for (int i = 0; i < 32; ++i) o[c * 32 + i] = f2bf(__uint_as_float(r[i]) / l);
    }
  }
};

}  // namespace

extern "C" __attribute__((visibility("default"))) int lost_copy(const void* q, const void* k, const void* v, void* out,
                                                                int items, int keys, int grid, int lost, int lost_item,
                                                                int lost_tile, unsigned* err, cudaStream_t stream) {
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, q, items * 2 * kTile, 64, 64) || !make_map(&mk, k, keys, 64, 64) || !make_map(&mv, v, keys, 64, 64))
    return -1;
  auto kernel = tc_items_kernel<Plain>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ItemsCfg<Plain>::SMEM) != cudaSuccess)
    return -2;
  const Plain p{static_cast<__nv_bfloat16*>(out), items, keys, 0.125f * 1.4426950408889634f, lost, lost_item, lost_tile};
  kernel<<<grid, kItemThreads, ItemsCfg<Plain>::SMEM, stream>>>(mq, mk, mv, p, err);
  return (int)cudaGetLastError();
}

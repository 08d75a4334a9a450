// Symmetric 8-bit quantisation of a bf16 row: scale = fp32(amax / 127), q = the
// integer nearest to 127 x / amax, ties to even.
//
// One FMA decides that integer exactly: x k + 1.5 2^23, whose single rounding is
// to an integer, ties to even (the low byte of the result), with k = 127 / amax.
// Write a, b for the 8-bit significands of amax and x, t = 127 b / (a 2^s):
//   a = 254 = 2 * 127: k is a power of two, so x k is exact and so are its ties;
//   otherwise (127 is prime) t is a half integer only where x = +-amax / 2, and
//   the even neighbour is +-64, the one away from zero: k raised by 2^-20 takes
//   it.  Any other t is at least 2^-s / 255 from a half integer, and raising k
//   and rounding it (3 ulp) move t by less than 127 2^-s (2^-20 + 2^-21.4) =
//   2^-s / 4600.
#pragma once

#include "common.cuh"

namespace b200 {

struct RowQuant {
  float unit;   // a power of two that takes amax into fp32's normal range
  float k;      // 127 / (amax unit), raised where that decides ties
  float scale;  // what a unit of q stands for (0: zero row, NaN: a non-finite row)
  bool zero;    // all q are 0
};

// From the row's largest |x| as bf16 bits (as integers they order like the
// magnitudes, infinity above all numbers and NaN above infinity).
B200_DEV RowQuant row_quant(uint32_t amax_bits) {
  RowQuant r;
  const float a = __uint_as_float(amax_bits << 16);
  const bool finite = amax_bits < 0x7f80u;
  r.zero = amax_bits == 0u || !finite;
  r.unit = a < 0x1p-100f ? 0x1p100f : 1.f;
  const bool power = (__float_as_uint(a * r.unit) >> 16 & 0x7fu) == 0x7eu;  // significand 254
  r.k = __fdiv_rn(127.f, a * r.unit) * (power ? 1.f : 1.f + 0x1p-20f);
  r.scale = finite ? __fdiv_rn(a, 127.f) : __int_as_float(0x7fffffff);
  return r;
}

// q in the low byte.
B200_DEV uint32_t quant1(float x, const RowQuant& r) { return __float_as_uint(fmaf(x * r.unit, r.k, 12582912.f)); }

// 8 bf16 values -> 8 bytes.
B200_DEV uint2 quant8(const uint4& u, const RowQuant& r) {
  if (r.zero) return make_uint2(0u, 0u);
  float f[8];
  unpack8(u, f);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = quant1(f[i], r);
  uint2 o;
  o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return o;
}

// Largest magnitudes (as bf16 bits) of packed pairs, both halves apart.
B200_DEV uint32_t amax_pairs(uint32_t m, const uint4& u) {
  m = __vmaxu2(m, u.x & 0x7fff7fffu);
  m = __vmaxu2(m, u.y & 0x7fff7fffu);
  m = __vmaxu2(m, u.z & 0x7fff7fffu);
  return __vmaxu2(m, u.w & 0x7fff7fffu);
}

// A warp's largest magnitude (bf16 bits) from every lane's packed pair.
B200_DEV uint32_t warp_amax(uint32_t m) { return __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16)); }

// The same over a block of NT threads; red: NT / 32 words of shared memory.
template <int NT>
B200_DEV uint32_t block_amax(uint32_t m, uint32_t* red) {
  m = warp_amax(m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) m = max(m, red[i]);
  return m;
}

}  // namespace b200

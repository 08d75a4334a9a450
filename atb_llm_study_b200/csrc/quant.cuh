// Symmetric 8-bit quantisation of a bf16 row: scale = fp32(amax / 127), q = the
// integer nearest to 127 x / amax, ties to even.
//
// The nearest integer is exact, not subject to the rounding of a quotient: for
// a bf16 x (8 significant bits) 127 x is exact in fp32, so is q amax, and so
// is the remainder e = 127 x - q amax (one FMA: both terms are multiples of
// 2^-7 ulp(x), and |e| stays below 2 amax).  A reciprocal product gives q to
// within one, and comparing 2|e| with amax settles it, ties included.
#pragma once

#include "common.cuh"

namespace b200 {

struct RowQuant {
  float mul;    // 127, times a power of two that keeps 127 x and 1 / amax inside fp32's range
  float amax;   // times the same power of two
  float inv;    // about 1 / amax
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
  const float c = a < 0x1p-100f ? 0x1p100f : (a > 0x1p100f ? 0x1p-30f : 1.f);
  r.mul = 127.f * c;
  r.amax = a * c;
  r.inv = __frcp_rn(r.amax);
  r.scale = finite ? __fdiv_rn(a, 127.f) : __int_as_float(0x7fffffff);
  return r;
}

B200_DEV int quant1(float x, const RowQuant& r) {
  const float p = x * r.mul;
  float q = rintf(p * r.inv);
  const float e = fmaf(-q, r.amax, p);
  const float e2 = 2.f * fabsf(e);
  int qi = (int)q;
  if (e2 > r.amax || (e2 == r.amax && (qi & 1))) qi += e > 0.f ? 1 : -1;
  return qi;
}

// 8 bf16 values -> 8 bytes.
B200_DEV uint2 quant8(const uint4& u, const RowQuant& r) {
  if (r.zero) return make_uint2(0u, 0u);
  float f[8];
  unpack8(u, f);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = (uint32_t)quant1(f[i], r);
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

// The block's largest magnitude (bf16 bits) from every thread's packed pair;
// red: NT / 32 words of shared memory, free again after the next __syncthreads.
template <int NT>
B200_DEV uint32_t block_amax(uint32_t m, uint32_t* red) {
  m = max(m & 0xffffu, m >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) m = max(m, red[i]);
  return m;
}

}  // namespace b200

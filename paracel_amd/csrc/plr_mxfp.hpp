// Device helpers shared by the 4-bit operators, dropout and the pass over a shard held in 4
// bits: the microscaled 4-bit format and the dropout mask.
//
// Format: 32 consecutive values of a row share a power of two 2^(s - 127), s an unsigned byte
// (255: the block holds a value that is not finite, and stands for NaN throughout); a value is
// a 4-bit code of sign, two exponent bits and a mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Two
// codes to a byte, the even column in the low half.
//
// Mask: column j of row i is kept where a 16-bit word reaches the threshold rint(rate * 65536);
// the word is number j % 8 of the 128 bits that Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) gives for the counter
// (j / 8, i low, i high, step) under the seed as key.  So a mask costs no memory and every
// kernel that needs it -- the pass forward, the pass back, any tile shape -- makes the same one.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace plr_mx {

constexpr int kBlockCols = 32;

typedef float v2f __attribute__((ext_vector_type(2)));

struct Mask {
  unsigned threshold;  // kept where the word >= threshold
  unsigned key0, key1, step;
  int64_t row0;  // added to the row numbers of the launch
};

__device__ __forceinline__ void philox_round(unsigned (&c)[4], unsigned k0, unsigned k1) {
  const uint64_t p = (uint64_t)c[0] * 0xD2511F53u, q = (uint64_t)c[2] * 0xCD9E8D57u;
  const unsigned c1 = c[1], c3 = c[3];
  c[0] = (unsigned)(q >> 32) ^ c1 ^ k0;
  c[1] = (unsigned)q;
  c[2] = (unsigned)(p >> 32) ^ c3 ^ k1;
  c[3] = (unsigned)p;
}

// The keep bits of columns 8 * group .. 8 * group + 7 of a row (bit b: column 8 * group + b).
__device__ __forceinline__ unsigned keep8(const Mask& m, int64_t row, unsigned group) {
  const uint64_t r = (uint64_t)(row + m.row0);
  unsigned c[4] = {group, (unsigned)r, (unsigned)(r >> 32), m.step};
  unsigned k0 = m.key0, k1 = m.key1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  unsigned bits = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bits |= ((c[w] & 0xffffu) >= m.threshold ? 1u : 0u) << (2 * w);
    bits |= ((c[w] >> 16) >= m.threshold ? 1u : 0u) << (2 * w + 1);
  }
  return bits;
}

// 2^(s - 127) for a scale byte below 255 (s = 0 is the subnormal 2^-127).
__device__ __forceinline__ float scale_value(unsigned s) {
  return __uint_as_float(s ? s << 23 : 0x00400000u);
}
__device__ __forceinline__ double scale_value_f64(unsigned s) {
  return __hiloint2double((int)((s + (1023 - 127)) << 20), 0);
}

// Values 2 * P and 2 * P + 1 of a word of eight codes, unscaled.
template <int P>
__device__ __forceinline__ v2f decode2(unsigned word) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, P);
}

}  // namespace plr_mx

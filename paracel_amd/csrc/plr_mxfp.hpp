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

constexpr unsigned kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;
constexpr unsigned kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

__device__ __forceinline__ unsigned xor3(unsigned a, unsigned b, unsigned c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// The generator's first two rounds split into what depends on the column group alone and on the
// row alone (half of the counter each): a kernel that meets a group in many rows, or a row in
// several groups, makes each part once, and eight rounds are left per 8 values.
struct MaskGroup {
  unsigned a, b, c;
};
struct MaskRow {
  unsigned a, b, c;
};
__device__ __forceinline__ MaskGroup mask_group(const Mask& m, unsigned group) {
  const uint64_t p = (uint64_t)group * kPhiloxM0;
  const uint64_t q = (uint64_t)((unsigned)(p >> 32) ^ m.step ^ m.key1) * kPhiloxM1;
  return {(unsigned)(q >> 32) ^ (m.key0 + kPhiloxW0), (unsigned)q, (unsigned)p};
}
__device__ __forceinline__ MaskRow mask_row(const Mask& m, int64_t row) {
  const uint64_t r = (uint64_t)row + (uint64_t)m.row0;
  const uint64_t q = (uint64_t)(unsigned)(r >> 32) * kPhiloxM1;
  const uint64_t p = (uint64_t)xor3((unsigned)(q >> 32), (unsigned)r, m.key0) * kPhiloxM0;
  return {(unsigned)q, (unsigned)(p >> 32) ^ (m.key1 + kPhiloxW1), (unsigned)p};
}

// The 8 values of a group in a row: halves w of the result hold 1 where values 2 w and 2 w + 1 are
// dropped.
struct DropWords {
  unsigned w[4];
};
__device__ __forceinline__ DropWords drop_words(const Mask& m, const MaskGroup& g, const MaskRow& r) {
  unsigned c0 = g.a ^ r.a, c1 = g.b, c2 = r.b ^ g.c, c3 = r.c;
#pragma unroll
  for (int i = 2; i < 10; ++i) {
    const uint64_t p = (uint64_t)c0 * kPhiloxM0, q = (uint64_t)c2 * kPhiloxM1;
    c0 = xor3((unsigned)(q >> 32), c1, m.key0 + (unsigned)i * kPhiloxW0);
    c2 = xor3((unsigned)(p >> 32), c3, m.key1 + (unsigned)i * kPhiloxW1);
    c1 = (unsigned)q;
    c3 = (unsigned)p;
  }
  // threshold - word, not below 0, is 0 where the value is kept; at most 1 of it marks a drop.  (As
  // instructions: from vector operations the compiler makes a comparison and a selection for
  // every half word.)
  const unsigned t = m.threshold | m.threshold << 16, one = 0x00010001u;
  auto drops = [&](unsigned w) {
    unsigned d;
    asm("v_pk_sub_u16 %0, %1, %2 clamp" : "=v"(d) : "s"(t), "v"(w));
    asm("v_pk_min_u16 %0, %1, %2" : "=v"(d) : "s"(one), "v"(d));
    return d;
  };
  return {{drops(c0), drops(c1), drops(c2), drops(c3)}};
}
// The same as one word: bit 4 i is 1 where value i is dropped.
__device__ __forceinline__ unsigned drop_marks(const Mask& m, const MaskGroup& g, const MaskRow& r) {
  const DropWords d = drop_words(m, g, r);
  // bytes 0 and 2 of each word hold a mark: the even values' go to the bytes of one word, the
  // odd ones' to another's
  const unsigned lo = __builtin_amdgcn_perm(d.w[1], d.w[0], 0x06020400u);  // 0.0 1.0 0.2 1.2
  const unsigned hi = __builtin_amdgcn_perm(d.w[3], d.w[2], 0x06020400u);
  const unsigned even = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  const unsigned odd = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
  return even | odd << 4;
}
// Two 16-bit values, the marked ones zeroed.
__device__ __forceinline__ unsigned zero_dropped(unsigned pair, unsigned marks) {
  unsigned m;
  asm("v_pk_sub_u16 %0, 0, %1" : "=v"(m) : "v"(marks));
  return pair & ~m;
}
// Nibble i is 0xF where value i is kept, 0 where it is dropped.
__device__ __forceinline__ unsigned kept_nibbles(unsigned marks) { return ~((marks << 4) - marks); }

__device__ __forceinline__ unsigned drop_marks(const Mask& m, int64_t row, unsigned group) {
  return drop_marks(m, mask_group(m, group), mask_row(m, row));
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

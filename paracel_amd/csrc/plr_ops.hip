// Operators on device matrices: quantisation to microscaled 4-bit floating point and back, the
// product of two such matrices, and dropout.  The entry points (include/plr.h) take device
// pointers and a stream, enqueue kernels and return; they allocate nothing and keep nothing
// between calls.
#include "../../include/plr.h"

#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "plr_internal.hpp"
#include "plr_matmul.hpp"
#include "plr_mxfp.hpp"

namespace {

using namespace plr_mx;

// ---------------------------------------------------------------- element types
template <typename T>
struct Elem;
template <>
struct Elem<double> {
  typedef double wide;  // what a value is worked on in
  static __device__ __forceinline__ double up(double v) { return v; }
  static __device__ __forceinline__ double down(double v) { return v; }
};
template <>
struct Elem<float> {
  typedef float wide;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<__bf16> {
  typedef float wide;
  static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }
};
template <>
struct Elem<_Float16> {
  typedef float wide;
  static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};

// V consecutive values, moved in words of 16 bytes whatever the row's alignment: the device's
// global loads and stores need none (rows of 4100 bfloat16 start on 8-byte boundaries).
template <typename T, int V>
struct Pack {
  T v[V];
};
typedef int v4w __attribute__((ext_vector_type(4), aligned(2)));
template <int N>
struct Words {
  v4w w[N];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_whole(const T* p) {
  constexpr int N = (int)sizeof(T) * V / 16;
  Words<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.w[i] = reinterpret_cast<const v4w*>(p)[i];
  return __builtin_bit_cast(Pack<T, V>, r);
}

// Columns c .. c + V of a row at p (p = the row's first value); those at `cols` and behind are 0.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p, int64_t c, int64_t cols) {
  Pack<T, V> r;
  if (c + V <= cols) {
    r = load_whole<T, V>(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = c + i < cols ? p[c + i] : T(0);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, int64_t c, int64_t cols, const Pack<T, V>& r) {
  if (c + V <= cols) {
    constexpr int N = (int)sizeof(T) * V / 16;
    const Words<N> w = __builtin_bit_cast(Words<N>, r);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<v4w*>(p + c)[i] = w.w[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < cols) p[c + i] = r.v[i];
  }
}

// How the 32 columns of a block lie over a quad's lanes: lane l takes P pieces of V = 16 bytes'
// worth of columns, piece i from column 32 / P * i + V * l on, so that a quad's load or store is 64
// consecutive bytes for every type (with 8 consecutive columns to a lane the 250000 x 512 doubles
// below took 247 us to codes, 250000 x 512 floats 141 us back).
template <typename T>
struct Piece {
  static constexpr int V = 16 / (int)sizeof(T), P = 8 / V;
  static __device__ __forceinline__ int column(int i, int l) { return 32 / P * i + V * l; }
};
template <int A, int B, int C, int D>
__device__ __forceinline__ unsigned quad_perm(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, A | B << 2 | C << 4 | D << 6, 0xf, 0xf, true);
}
// Four codewords of a quad, byte b of lane l's to byte l of lane b's.
__device__ __forceinline__ unsigned quad_transpose(unsigned w, int l) {
  unsigned o = quad_perm<1, 0, 3, 2>(w);
  w = __builtin_amdgcn_perm(o, w, l & 1 ? 0x03070105u : 0x06020400u);
  o = quad_perm<2, 3, 0, 1>(w);
  return __builtin_amdgcn_perm(o, w, l & 2 ? 0x03020706u : 0x05040100u);
}
// A lane's 8 codes in the order of its pieces -> the codes of columns 8 l .. 8 l + 7, and back.
template <typename T>
__device__ __forceinline__ unsigned codes_in_order(unsigned w, int l) {
  if constexpr (Piece<T>::P == 1) return w;
  if constexpr (Piece<T>::P == 4) return quad_transpose(w, l);
  return __builtin_amdgcn_perm(quad_perm<1, 3, 1, 3>(w), quad_perm<0, 2, 0, 2>(w), l & 2 ? 0x07060302u : 0x05040100u);
}
template <typename T>
__device__ __forceinline__ unsigned codes_of_pieces(unsigned w, int l) {
  if constexpr (Piece<T>::P == 1) return w;
  if constexpr (Piece<T>::P == 4) return quad_transpose(w, l);
  return __builtin_amdgcn_perm(quad_perm<2, 2, 3, 3>(w), quad_perm<0, 0, 1, 1>(w), l & 1 ? 0x07060302u : 0x05040100u);
}
// The marks of columns 8 l .. 8 l + 7 (four bits each) -> those of the lane's pieces.
template <typename T>
__device__ __forceinline__ unsigned marks_of_pieces(unsigned m, int l) {
  if constexpr (Piece<T>::P == 1) return m;
  if constexpr (Piece<T>::P == 2)
    return (quad_perm<0, 0, 1, 1>(m) >> 16 * (l & 1) & 0xffffu) | quad_perm<2, 2, 3, 3>(m) >> 16 * (l & 1) << 16;
  return quad_transpose(m, l);
}
template <typename T>
__device__ __forceinline__ Pack<T, 8> load_pieces(const T* row, int64_t block, int l, int64_t cols) {
  Pack<T, 8> r;
#pragma unroll
  for (int i = 0; i < Piece<T>::P; ++i) {
    const auto p = load_pack<T, Piece<T>::V>(row, block + Piece<T>::column(i, l), cols);
#pragma unroll
    for (int e = 0; e < Piece<T>::V; ++e) r.v[Piece<T>::V * i + e] = p.v[e];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pieces(T* row, int64_t block, int l, int64_t cols, const Pack<T, 8>& r) {
#pragma unroll
  for (int i = 0; i < Piece<T>::P; ++i) {
    Pack<T, Piece<T>::V> p;
#pragma unroll
    for (int e = 0; e < Piece<T>::V; ++e) p.v[e] = r.v[Piece<T>::V * i + e];
    store_pack<T, Piece<T>::V>(row, block + Piece<T>::column(i, l), cols, p);
  }
}

// ---------------------------------------------------------------- quantisation
// The bits of |v| that order magnitudes and hold the exponent: for doubles the high word.
__device__ __forceinline__ unsigned mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned mag_bits(double v) {
  return (unsigned)__double2hiint(v) & 0x7fffffffu;
}
// Scale byte of a block from the largest mag_bits: floor(log2 max) - 2 (6 = 1.5 * 2^2 is the
// largest code), biased by 127, at least 0; 255 when a value is not finite.  NaN and infinity
// order above every finite value, so one maximum finds them too.
__device__ __forceinline__ unsigned scale_byte(unsigned top, float) {
  const unsigned e = top >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ unsigned scale_byte(unsigned top, double) {
  const int e = (int)(top >> 20);
  if (e == 2047) return 255u;
  const int s = e - 1023 - 2 + 127;
  return (unsigned)(s < 0 ? 0 : s > 254 ? 254 : s);
}

// Eight values to eight codes, nearest with ties to the even code, saturating at 6.
__device__ __forceinline__ unsigned encode8(const float (&v)[8], unsigned s) {
  const float sc = scale_value(s);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
  return w;
}
// Doubles are scaled, then cut to a float's 24 bits with a last bit that says whether anything
// was cut off: the one rounding to four bits then goes the way the double's own would (a plain
// conversion to float could land on a tie the double is not on).
__device__ __forceinline__ float sticky_float(double v) {
  const int hi = __double2hiint(v);
  unsigned lo = (unsigned)__double2loint(v);
  lo = (lo & 0xe0000000u) | ((lo & 0x1fffffffu) ? 0x20000000u : 0u);
  return (float)__hiloint2double(hi, (int)lo);
}
__device__ __forceinline__ unsigned encode8(const double (&v)[8], unsigned s) {
  // 2^-(s - 127); doubles far outside a float's range meet s = 254 or s = 0 and saturate or vanish
  const double inv = __hiloint2double((int)((1023u + 127u - s) << 20), 0);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = sticky_float(fmin(fmax(v[i] * inv, -8.), 8.));
  return encode8(f, 127u);
}

// Pairs of 16-bit values are worked on as they lie, two to a word.
template <typename T>
constexpr bool kPairs = sizeof(T) == 2;
template <typename T, int SEL>
__device__ __forceinline__ unsigned encode_pair(unsigned old, unsigned pair, float sc) {
  if constexpr (std::is_same<T, __bf16>::value) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(v2, pair), sc, SEL);
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(v2, pair), sc, SEL);
  }
}
template <typename T>
__device__ __forceinline__ unsigned encode_pairs(const unsigned (&w)[4], float sc) {
  unsigned r = 0;
  r = encode_pair<T, 0>(r, w[0], sc);
  r = encode_pair<T, 1>(r, w[1], sc);
  r = encode_pair<T, 2>(r, w[2], sc);
  return encode_pair<T, 3>(r, w[3], sc);
}
// Larger magnitude of each half; the maximum so far is without signs.
__device__ __forceinline__ unsigned pair_max(unsigned top, unsigned pair) {
  unsigned r;
  asm("v_pk_max_u16 %0, %1, %2" : "=v"(r) : "v"(top), "v"(pair & 0x7fff7fffu));
  return r;
}
// mag_bits of the float that a 16-bit magnitude stands for.
template <typename T>
__device__ __forceinline__ unsigned half_mag_bits(unsigned half) {
  if constexpr (std::is_same<T, __bf16>::value) return half << 16;
  return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)half));
}

struct QuantArgs {
  const void* x;
  int64_t n, d, ldx;
  uint8_t* codes;
  int64_t ldc;
  uint8_t* scales;
  int64_t lds;
  int64_t chunks;  // 128-column chunks of an output row that are written
  int tc_log2;     // a workgroup's tile is 2^tc_log2 chunks wide
  unsigned nbx;    // tiles across
  Mask mask;
};

constexpr int kQuantThreads = 256;
// row sets per workgroup: few stores to a thread keep more of them going at once (250000 x 512
// floats to codes and back: 99 + 120 us with one set, 106 + 142 with four), but the mask's first
// rounds and narrow loads want a few (16385 x 4100 bfloat16: 28 and 28 us with three and two, 32 and
// 28 with one)
template <typename T>
constexpr int kQuantRows = sizeof(T) == 2 ? 3 : 1;
template <typename T>
constexpr int kMoveRows = sizeof(T) == 2 ? 2 : 1;
// waves of a workgroup of quantize_columns, side by side along the rows of x: unaligned rows have
// lines that two of them read (16385 x 4100 bfloat16: 49 us with one, 38 with four, 42 with eight)
constexpr int kColumnWaves = 4;

// Largest of the four lanes of a quad, in all four.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);  // lanes 1 0 3 2
  v = v > o ? v : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);  // lanes 2 3 0 1
  return v > o ? v : o;
}

// Blocks along a row.  A thread takes 8 columns, a quad a block, 16 lanes a chunk of 128 columns;
// the workgroup's 16 chunk slots are 2^tc across and 16 / 2^tc rows.  Bound by the bytes of x:
// 250000 x 512 doubles 190 us call after call, 5.7 TB/s (233 in turn with the way back to floats);
// 16385 x 4100 bfloat16 28 us, 6.2 TB/s, with dropout 44 (there by the generator's 60 instructions per
// 8 values).
template <typename T, bool DROP>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows(QuantArgs a) {
  typedef typename Elem<T>::wide W;
  const unsigned by = blockIdx.x / a.nbx, bx = blockIdx.x - by * a.nbx;
  const int slot = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const int64_t chunk = ((int64_t)bx << a.tc_log2) + (slot & ((1 << a.tc_log2) - 1));
  const int rows = 16 >> a.tc_log2;  // rows per set
  const int64_t row = (int64_t)by * rows * kQuantRows<T> + (slot >> a.tc_log2);
  const int64_t c = chunk * 128 + l16 * 8, block = c & ~31;
  const int l4 = l16 & 3;
  const T* x = static_cast<const T*>(a.x);
  const MaskGroup group = DROP ? mask_group(a.mask, (unsigned)(c >> 3)) : MaskGroup{};
  Pack<T, 8> in[kQuantRows<T>];
#pragma unroll
  for (int u = 0; u < kQuantRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r < a.n) in[u] = load_pieces<T>(x + r * a.ldx, block, l4, a.d);
  }
#pragma unroll
  for (int u = 0; u < kQuantRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r >= a.n) continue;  // (a quad shares its row: its lanes leave together)
    unsigned top = 0, s, w;
    if constexpr (kPairs<T>) {
      v4w raw = __builtin_bit_cast(v4w, in[u]);
      unsigned pairs[4] = {(unsigned)raw.x, (unsigned)raw.y, (unsigned)raw.z, (unsigned)raw.w};
      if (DROP) {
        const DropWords d = drop_words(a.mask, group, mask_row(a.mask, r));
#pragma unroll
        for (int i = 0; i < 4; ++i) pairs[i] = zero_dropped(pairs[i], d.w[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) top = pair_max(top, pairs[i]);
      top = (top & 0xffffu) > top >> 16 ? top & 0xffffu : top >> 16;
      s = scale_byte(half_mag_bits<T>(quad_max(top)), 0.f);
      w = s == 255u ? 0u : encode_pairs<T>(pairs, scale_value(s));
    } else {
      W v[8];
      const unsigned drop = DROP ? marks_of_pieces<T>(drop_marks(a.mask, group, mask_row(a.mask, r)), l4) : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = Elem<T>::up(in[u].v[i]);
        if (DROP && (drop >> 4 * i & 1)) v[i] = W(0);
        const unsigned b = mag_bits(v[i]);
        top = b > top ? b : top;
      }
      s = scale_byte(quad_max(top), W(0));
      w = codes_in_order<T>(s == 255u ? 0u : encode8(v, s), l4);
    }
    if (c / 2 < a.ldc && chunk < a.chunks)
      *reinterpret_cast<unsigned*>(a.codes + r * a.ldc + c / 2) = w;
    if ((l16 & 3) == 0 && c / 32 < a.lds && chunk < a.chunks)
      a.scales[r * a.lds + c / 32] = (uint8_t)s;
  }
}

// 32 values of one column, V columns of them in `in`, to a block of the result's row `j`.
template <typename T, int V>
__device__ __forceinline__ void put_column_block(const QuantArgs& a, const Pack<T, V> (&in)[32], int k, int64_t j,
                                                 int64_t blk) {
  typedef typename Elem<T>::wide W;
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const unsigned b = mag_bits(Elem<T>::up(in[i].v[k]));
    top = b > top ? b : top;
  }
  const unsigned s = scale_byte(top, W(0));
  uint4 w;
  unsigned* ww = reinterpret_cast<unsigned*>(&w);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    W v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<T>::up(in[8 * q + i].v[k]);
    ww[q] = s == 255u ? 0u : encode8(v, s);
  }
  *reinterpret_cast<uint4*>(a.codes + j * a.ldc + blk * 16) = w;
  if (blk < a.lds) a.scales[j * a.lds + blk] = (uint8_t)s;
}

// Blocks along a column: row j of the result is column j of x.  A thread holds V = 16 bytes of
// columns times 32 rows in registers -- so a block never leaves its thread --, 8 lanes cover 128
// bytes of a row of x and the 8 groups of lanes 256 rows, so that a result row is written in
// pieces of 128 bytes.  The columns behind the last whole V are left to a wave of their own (the
// last of a tile row), where a thread takes one column.  250000 x 512 doubles 211 us, 5.2 TB/s;
// 16385 x 4100 bfloat16 38 us, with dropout 40 (48 in turn with the way back): two waves to a SIMD,
// their tiles fill the registers.
template <typename T, bool DROP>
__global__ __launch_bounds__(64 * kColumnWaves, 2) void quantize_columns(QuantArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  const unsigned by = blockIdx.x / a.nbx;
  const unsigned bx = (blockIdx.x - by * a.nbx) * kColumnWaves + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t blk = (int64_t)by * 8 + (lane >> 3);  // block of 32 rows
  const int64_t r0 = blk * 32;
  const int64_t whole = a.d / V * V;
  if (blk * 16 >= a.ldc || blk >= a.chunks * 4) return;
  const T* x = static_cast<const T*>(a.x);
  if ((int64_t)bx * 8 * V >= whole) {
    if ((int64_t)bx * 8 * V >= whole + 8 * V) return;  // one wave for what is over
    const int64_t c = whole + (lane & 7);
    if (c >= a.d) return;
    const MaskGroup group = DROP ? mask_group(a.mask, (unsigned)(c >> 3)) : MaskGroup{};
    Pack<T, 1> in[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      in[i].v[0] = r0 + i < a.n ? x[(r0 + i) * a.ldx + c] : T(0);
      if (DROP && (drop_marks(a.mask, group, mask_row(a.mask, r0 + i)) >> 4 * (c & 7) & 1)) in[i].v[0] = T(0);
    }
    put_column_block<T, 1>(a, in, 0, c, blk);
    return;
  }
  const int64_t c0 = ((int64_t)bx * 8 + (lane & 7)) * V;  // first column of x
  if (c0 >= whole) return;
  const Pack<T, V> zero = {};
  Pack<T, V> in[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    // rows behind the last one repeat it here and are zeroed below
    const int64_t r = r0 + i < a.n ? r0 + i : a.n - 1;
    in[i] = load_whole<T, V>(x + r * a.ldx + c0);
  }
  if (r0 + 32 > a.n) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (r0 + i >= a.n) in[i] = zero;
  }
  if constexpr (kPairs<T>) {
    // two columns at a time: both maxima in one word, then pairs of rows of either column
    v4w raw[32];
    const MaskGroup group = DROP ? mask_group(a.mask, (unsigned)(c0 >> 3)) : MaskGroup{};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      raw[i] = __builtin_bit_cast(v4w, in[i]);
      if (DROP) {
        const DropWords d = drop_words(a.mask, group, mask_row(a.mask, r0 + i));
#pragma unroll
        for (int k = 0; k < 4; ++k) raw[i][k] = (int)zero_dropped((unsigned)raw[i][k], d.w[k]);
        // row after row: 32 generator calls at once take more registers than there are
        asm volatile("" : "+v"(raw[i]));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = pair_max(top, (unsigned)raw[i][k]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned s = scale_byte(half_mag_bits<T>(h ? top >> 16 : top & 0xffffu), 0.f);
        const float sc = scale_value(s);
        uint4 w = uint4{0, 0, 0, 0};
        if (s != 255u) {
          unsigned* ww = reinterpret_cast<unsigned*>(&w);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            unsigned pairs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              pairs[i] = __builtin_amdgcn_perm((unsigned)raw[8 * q + 2 * i + 1][k], (unsigned)raw[8 * q + 2 * i][k],
                                               h ? 0x07060302u : 0x05040100u);
            ww[q] = encode_pairs<T>(pairs, sc);
          }
        }
        const int64_t j = c0 + 2 * k + h;
        *reinterpret_cast<uint4*>(a.codes + j * a.ldc + blk * 16) = w;
        if (blk < a.lds) a.scales[j * a.lds + blk] = (uint8_t)s;
      }
    }
    return;
  }
  if (DROP) {
    const MaskGroup group = mask_group(a.mask, (unsigned)(c0 >> 3));
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const unsigned drop = drop_marks(a.mask, group, mask_row(a.mask, r0 + i)) >> 4 * (c0 & 7);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (drop >> 4 * k & 1) in[i].v[k] = T(0);
        asm volatile("" : "+v"(in[i].v[k]));
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) put_column_block<T, V>(a, in, k, c0 + k, blk);
}

struct DequantArgs {
  const uint8_t* codes;
  int64_t ldc;
  const uint8_t* scales;
  int64_t lds;
  void* out;
  int64_t n, d, ldo;
  int tc_log2;
  unsigned nbx;
};

// The same layout the other way: a lane loads the codes of 8 columns, the quad deals them out.  Bound
// by the bytes written: 250000 x 512 floats 115 to 120 us, 4.8 to 5.0 TB/s (a fill alone 6.9, a copy 5.1).
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void dequantize_rows(DequantArgs a) {
  typedef typename Elem<T>::wide W;
  const unsigned by = blockIdx.x / a.nbx, bx = blockIdx.x - by * a.nbx;
  const int slot = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const int64_t chunk = ((int64_t)bx << a.tc_log2) + (slot & ((1 << a.tc_log2) - 1));
  const int rows = 16 >> a.tc_log2;
  const int64_t row = (int64_t)by * rows * kMoveRows<T> + (slot >> a.tc_log2);
  const int64_t c = chunk * 128 + l16 * 8, block = c & ~31;
  const int l4 = l16 & 3;
  if (block >= a.d) return;  // (a quad's lanes stay together; a started block has all its codes)
  unsigned w[kMoveRows<T>], s[kMoveRows<T>];
#pragma unroll
  for (int u = 0; u < kMoveRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r < a.n) {
      w[u] = *reinterpret_cast<const unsigned*>(a.codes + r * a.ldc + c / 2);
      s[u] = a.scales[r * a.lds + c / 32];
    }
  }
#pragma unroll
  for (int u = 0; u < kMoveRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r >= a.n) continue;
    // the product with the scale is exact in the wide type unless it leaves its range
    const unsigned wp = codes_of_pieces<T>(w[u], l4);
    const v2f q[4] = {decode2<0>(wp), decode2<1>(wp), decode2<2>(wp), decode2<3>(wp)};
    const W sc = s[u] == 255u ? W(__builtin_nanf("")) : sizeof(W) == 8 ? W(scale_value_f64(s[u]))
                                                                       : W(scale_value(s[u]));
    Pack<T, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = Elem<T>::down((W)q[i >> 1][i & 1] * sc);
    store_pieces<T>(static_cast<T*>(a.out) + r * a.ldo, block, l4, a.d, o);
  }
}

// ---------------------------------------------------------------- dropout
struct DropArgs {
  const void* x;
  void* out;
  int64_t n, d, ldx, ldo;
  int tc_log2;
  unsigned nbx;
  double scale;
  Mask mask;
};

// A thread takes 8 values, one generator call; bound by the bytes moved: 32768 x 8192 bfloat16 182 us,
// 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void dropout_rows(DropArgs a) {
  typedef typename Elem<T>::wide W;
  const unsigned by = blockIdx.x / a.nbx, bx = blockIdx.x - by * a.nbx;
  const int slot = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const int64_t chunk = ((int64_t)bx << a.tc_log2) + (slot & ((1 << a.tc_log2) - 1));
  const int rows = 16 >> a.tc_log2;
  const int64_t row = (int64_t)by * rows * kMoveRows<T> + (slot >> a.tc_log2);
  const int64_t c = chunk * 128 + l16 * 8, block = c & ~31;
  const int l4 = l16 & 3;
  if (block >= a.d) return;  // (a quad's lanes stay together)
  Pack<T, 8> in[kMoveRows<T>];
#pragma unroll
  for (int u = 0; u < kMoveRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r < a.n) in[u] = load_pieces<T>(static_cast<const T*>(a.x) + r * a.ldx, block, l4, a.d);
  }
  const W sc = (W)a.scale;
  const MaskGroup group = mask_group(a.mask, (unsigned)(c >> 3));
#pragma unroll
  for (int u = 0; u < kMoveRows<T>; ++u) {
    const int64_t r = row + (int64_t)u * rows;
    if (r >= a.n) continue;
    const unsigned drop = marks_of_pieces<T>(drop_marks(a.mask, group, mask_row(a.mask, r)), l4);
    Pack<T, 8> o;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      o.v[i] = (drop >> 4 * i & 1) ? T(0) : Elem<T>::down(Elem<T>::up(in[u].v[i]) * sc);
    store_pieces<T>(static_cast<T*>(a.out) + r * a.ldo, block, l4, a.d, o);
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxDevices = 64;
std::atomic<int> g_cu[kMaxDevices];  // compute units of a checked gfx950 device, 0: not looked at

int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }

// One call: the caller's current device is left as it was found, failures are recorded under the
// entry point's name.
struct Call {
  const char* name;
  int prev = -1;
  hipStream_t stream = nullptr;
  int cus = 0;
  explicit Call(const char* entry) : name(entry) {}
  ~Call() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
  int bad(int code, const char* what) const {
    char b[256];
    snprintf(b, sizeof b, "%s: %s", name, what);
    return plr_fail_without_context(code, b);
  }
  int hip(hipError_t e, const char* what) const {
    char b[256];
    (void)hipGetLastError();
    snprintf(b, sizeof b, "%s: %s failed: %s", name, what, hipGetErrorString(e));
    return plr_fail_without_context(e == hipErrorOutOfMemory ? PLR_ERR_NOMEM : PLR_ERR_HIP, b);
  }
  int begin(int device_id, void* hip_stream) {
    stream = reinterpret_cast<hipStream_t>(hip_stream);
    if (device_id < 0 || device_id >= kMaxDevices)
      return bad(PLR_ERR_INVALID, "device_id out of range");
    (void)hipGetLastError();  // what the caller left behind is not this call's (launched())
    int cur = -1;
    hipError_t e = hipGetDevice(&cur);
    if (e != hipSuccess) return hip(e, "hipGetDevice");
    if (cur != device_id) {
      if ((e = hipSetDevice(device_id)) != hipSuccess) return hip(e, "hipSetDevice");
      prev = cur;
    }
    cus = g_cu[device_id].load();
    if (cus == 0) {
      // once per device; not stream work, so a caller that captures makes one call before
      hipDeviceProp_t prop;
      if ((e = hipGetDeviceProperties(&prop, device_id)) != hipSuccess)
        return hip(e, "hipGetDeviceProperties");
      if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
        return bad(PLR_ERR_UNSUPPORTED, "this library carries gfx950 code only");
      cus = prop.multiProcessorCount;
      g_cu[device_id].store(cus);
    }
    return PLR_OK;
  }
  int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? (int)PLR_OK : hip(e, "launch");
  }
};

size_t type_size(unsigned t) {
  switch (t) {
    case PLR_F64: return 8;
    case PLR_F32: return 4;
    case PLR_BF16:
    case PLR_F16: return 2;
  }
  return 0;
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
// rows * pitch elements of `size` bytes can be addressed
bool fits(int64_t rows, int64_t pitch, size_t size) {
  return rows == 0 || pitch <= INT64_MAX / (int64_t)size / rows;
}

int check_mask(Call& c, const plr_dropout* drop, Mask* m, double* scale) {
  *m = Mask{0, 0, 0, 0, 0};
  *scale = 1.;
  if (!drop) return PLR_OK;
  if (!(drop->rate >= 0. && drop->rate < 1.))
    return c.bad(PLR_ERR_INVALID, "dropout rate must be at least 0 and below 1");
  const unsigned t = (unsigned)rint(drop->rate * 65536.);
  if (t > 65535u)
    return c.bad(PLR_ERR_INVALID, "dropout rate must be at most 65535/65536");
  if (drop->row0 < 0) return c.bad(PLR_ERR_INVALID, "dropout row0 must be >= 0");
  m->threshold = t;
  m->key0 = (unsigned)drop->seed;
  m->key1 = (unsigned)(drop->seed >> 32);
  m->step = drop->step;
  m->row0 = drop->row0;
  *scale = 65536. / (65536. - t);
  return PLR_OK;
}

// Tiles of 16 chunk slots: as wide as the row needs, at most 16 chunks.
int tile_log2(int64_t chunks) {
  int t = 0;
  while (t < 4 && (int64_t)(1 << t) < chunks) ++t;
  return t;
}

// A launch counts its threads in 32 bits.
bool fits_launch(int64_t x, int64_t y, int threads) {
  return y == 0 || x <= (int64_t)0xffffffffu / threads / y;
}

// The tiled kernels over n rows of `chunks` chunks: launch(first row, rows, tiles across, grid) for
// as many rows at a time as a launch holds.
template <typename F>
void over_rows(int64_t n, int64_t chunks, int tc, int sets, F launch) {
  const int64_t tile = (int64_t)(16 >> tc) * sets;
  const int64_t x = ceil_div(chunks, (int64_t)1 << tc);  // at most 2^23
  const int64_t most = (int64_t)0xffffffffu / kQuantThreads / x * tile;
  for (int64_t r0 = 0; r0 < n; r0 += most) {
    const int64_t rows = std::min(most, n - r0);
    launch(r0, rows, (unsigned)x, (unsigned)(x * ceil_div(rows, tile)));
  }
}

template <typename T>
void launch_quantize(QuantArgs a, bool transpose, bool drop, unsigned grid, hipStream_t st) {
  if (transpose) {
    auto f = drop ? quantize_columns<T, true> : quantize_columns<T, false>;
    hipLaunchKernelGGL(f, dim3(grid), dim3(64 * kColumnWaves), 0, st, a);
  } else {
    auto f = drop ? quantize_rows<T, true> : quantize_rows<T, false>;
    a.tc_log2 = tile_log2(a.chunks);
    over_rows(a.n, a.chunks, a.tc_log2, kQuantRows<T>, [&](int64_t r0, int64_t rows, unsigned x, unsigned g) {
      QuantArgs b = a;
      b.x = static_cast<const T*>(a.x) + r0 * a.ldx;
      b.codes += r0 * a.ldc;
      b.scales += r0 * a.lds;
      b.mask.row0 = (int64_t)((uint64_t)a.mask.row0 + (uint64_t)r0);
      b.n = rows;
      b.nbx = x;
      hipLaunchKernelGGL(f, dim3(g), dim3(kQuantThreads), 0, st, b);
    });
  }
}

template <typename T>
void launch_dequantize(DequantArgs a, hipStream_t st) {
  const int64_t chunks = ceil_div(a.d, 128);
  a.tc_log2 = tile_log2(chunks);
  over_rows(a.n, chunks, a.tc_log2, kMoveRows<T>, [&](int64_t r0, int64_t rows, unsigned x, unsigned g) {
    DequantArgs b = a;
    b.codes += r0 * a.ldc;
    b.scales += r0 * a.lds;
    b.out = static_cast<T*>(a.out) + r0 * a.ldo;
    b.n = rows;
    b.nbx = x;
    hipLaunchKernelGGL(dequantize_rows<T>, dim3(g), dim3(kQuantThreads), 0, st, b);
  });
}

template <typename T>
void launch_dropout(DropArgs a, hipStream_t st) {
  const int64_t chunks = ceil_div(a.d, 128);
  a.tc_log2 = tile_log2(chunks);
  over_rows(a.n, chunks, a.tc_log2, kMoveRows<T>, [&](int64_t r0, int64_t rows, unsigned x, unsigned g) {
    DropArgs b = a;
    b.x = static_cast<const T*>(a.x) + r0 * a.ldx;
    b.out = static_cast<T*>(a.out) + r0 * a.ldo;
    b.mask.row0 = (int64_t)((uint64_t)a.mask.row0 + (uint64_t)r0);
    b.n = rows;
    b.nbx = x;
    hipLaunchKernelGGL(dropout_rows<T>, dim3(g), dim3(kQuantThreads), 0, st, b);
  });
}

}  // namespace

extern "C" {

int64_t plr_mxfp_code_pitch(int64_t d) { return d < 1 || d > INT64_MAX - 128 ? 0 : ceil_div(d, 128) * 64; }
int64_t plr_mxfp_scale_pitch(int64_t d) { return d < 1 || d > INT64_MAX - 128 ? 0 : ceil_div(d, 128) * 4; }

int plr_mxfp_quantize(int device_id, void* hip_stream, const void* dx, unsigned type, int64_t n,
                      int64_t d, int64_t ldx, unsigned flags, const plr_dropout* drop,
                      uint8_t* dcodes, int64_t ldc, uint8_t* dscales, int64_t lds) {
  Call c("plr_mxfp_quantize");
  const size_t size = type_size(type);
  if (size == 0) return c.bad(PLR_ERR_INVALID, "unknown element type");
  if (flags & ~(unsigned)PLR_MXFP_TRANSPOSE) return c.bad(PLR_ERR_INVALID, "unknown flag");
  if (n < 0 || d < 1) return c.bad(PLR_ERR_INVALID, "need n >= 0 and d >= 1");
  if (ldx < d) return c.bad(PLR_ERR_INVALID, "ldx must be >= d");
  const bool tr = (flags & PLR_MXFP_TRANSPOSE) != 0;
  const int64_t rows = tr ? d : n, cols = tr ? n : d;  // of the result
  if (d > (int64_t)1 << 34 || (tr && n > (int64_t)1 << 34))
    return c.bad(PLR_ERR_INVALID, "a row of more than 2^34 values");
  const int64_t blocks = ceil_div(cols, kBlockCols);
  if (ldc % 16 != 0 || ldc < blocks * 16)
    return c.bad(PLR_ERR_INVALID, "code pitch must be a multiple of 16 and hold the row's blocks of 16 bytes");
  if (lds < blocks) return c.bad(PLR_ERR_INVALID, "scale pitch must hold a byte per block of 32 columns");
  if (!fits(n, ldx, size) || !fits(rows, ldc, 1) || !fits(rows, lds, 1))
    return c.bad(PLR_ERR_INVALID, "matrix too large to address");
  Mask mask;
  double scale;
  int rc = check_mask(c, drop, &mask, &scale);
  if (rc != PLR_OK) return rc;
  if (n > 0 && (!dx || !dcodes || !dscales))
    return c.bad(PLR_ERR_INVALID, "device pointers must not be NULL");
  if (!aligned(dx, size)) return c.bad(PLR_ERR_INVALID, "dx must be aligned to its element type");
  if (!aligned(dcodes, 16)) return c.bad(PLR_ERR_INVALID, "dcodes must be 16-byte aligned");
  QuantArgs a;
  a.x = dx;
  a.n = n;
  a.d = d;
  a.ldx = ldx;
  a.codes = dcodes;
  a.ldc = ldc;
  a.scales = dscales;
  a.lds = lds;
  // whole 128-column chunks are written as far as the pitches reach
  a.chunks = ceil_div(cols, 128);
  a.mask = mask;
  a.tc_log2 = 0;
  unsigned grid = 0;
  if (tr) {
    const int64_t v = 16 / (int64_t)size;  // columns a thread takes; what is over has its own waves
    const int64_t x = ceil_div(ceil_div(d / v, 8) + (d % v != 0), kColumnWaves), y = ceil_div(a.chunks * 4, 8);
    if (!fits_launch(x, y, 64 * kColumnWaves)) return c.bad(PLR_ERR_INVALID, "matrix too large for one launch");
    a.nbx = (unsigned)x;
    grid = (unsigned)(x * y);
  }
  rc = c.begin(device_id, hip_stream);
  if (rc != PLR_OK || n == 0) return rc;
  const bool dr = drop != nullptr && mask.threshold > 0;
  switch (type) {
    case PLR_F64: launch_quantize<double>(a, tr, dr, grid, c.stream); break;
    case PLR_F32: launch_quantize<float>(a, tr, dr, grid, c.stream); break;
    case PLR_BF16: launch_quantize<__bf16>(a, tr, dr, grid, c.stream); break;
    default: launch_quantize<_Float16>(a, tr, dr, grid, c.stream); break;
  }
  return c.launched();
}

int plr_mxfp_dequantize(int device_id, void* hip_stream, const uint8_t* dcodes, int64_t ldc,
                        const uint8_t* dscales, int64_t lds, int64_t n, int64_t d, void* dout,
                        unsigned type, int64_t ldo) {
  Call c("plr_mxfp_dequantize");
  const size_t size = type_size(type);
  if (size == 0) return c.bad(PLR_ERR_INVALID, "unknown element type");
  if (n < 0 || d < 1) return c.bad(PLR_ERR_INVALID, "need n >= 0 and d >= 1");
  if (d > (int64_t)1 << 34) return c.bad(PLR_ERR_INVALID, "a row of more than 2^34 values");
  if (ldo < d) return c.bad(PLR_ERR_INVALID, "ldo must be >= d");
  const int64_t blocks = ceil_div(d, kBlockCols);
  if (ldc % 16 != 0 || ldc < blocks * 16)
    return c.bad(PLR_ERR_INVALID, "code pitch must be a multiple of 16 and hold the row's blocks of 16 bytes");
  if (lds < blocks) return c.bad(PLR_ERR_INVALID, "scale pitch must hold a byte per block of 32 columns");
  if (!fits(n, ldo, size) || !fits(n, ldc, 1) || !fits(n, lds, 1))
    return c.bad(PLR_ERR_INVALID, "matrix too large to address");
  if (n > 0 && (!dout || !dcodes || !dscales))
    return c.bad(PLR_ERR_INVALID, "device pointers must not be NULL");
  if (!aligned(dout, size)) return c.bad(PLR_ERR_INVALID, "dout must be aligned to its element type");
  if (!aligned(dcodes, 16)) return c.bad(PLR_ERR_INVALID, "dcodes must be 16-byte aligned");
  DequantArgs a;
  a.codes = dcodes;
  a.ldc = ldc;
  a.scales = dscales;
  a.lds = lds;
  a.out = dout;
  a.n = n;
  a.d = d;
  a.ldo = ldo;
  int rc = c.begin(device_id, hip_stream);
  if (rc != PLR_OK || n == 0) return rc;
  switch (type) {
    case PLR_F64: launch_dequantize<double>(a, c.stream); break;
    case PLR_F32: launch_dequantize<float>(a, c.stream); break;
    case PLR_BF16: launch_dequantize<__bf16>(a, c.stream); break;
    default: launch_dequantize<_Float16>(a, c.stream); break;
  }
  return c.launched();
}

int plr_dropout_apply(int device_id, void* hip_stream, const void* dx, unsigned type, int64_t n,
                      int64_t d, int64_t ldx, void* dout, int64_t ldo, const plr_dropout* drop) {
  Call c("plr_dropout_apply");
  const size_t size = type_size(type);
  if (size == 0) return c.bad(PLR_ERR_INVALID, "unknown element type");
  if (n < 0 || d < 1) return c.bad(PLR_ERR_INVALID, "need n >= 0 and d >= 1");
  if (d > (int64_t)1 << 34) return c.bad(PLR_ERR_INVALID, "a row of more than 2^34 values");
  if (ldx < d || ldo < d) return c.bad(PLR_ERR_INVALID, "ldx and ldo must be >= d");
  if (!fits(n, ldx, size) || !fits(n, ldo, size))
    return c.bad(PLR_ERR_INVALID, "matrix too large to address");
  if (!drop) return c.bad(PLR_ERR_INVALID, "drop must not be NULL");
  DropArgs a;
  int rc = check_mask(c, drop, &a.mask, &a.scale);
  if (rc != PLR_OK) return rc;
  if (n > 0 && (!dx || !dout)) return c.bad(PLR_ERR_INVALID, "device pointers must not be NULL");
  if (!aligned(dx, size) || !aligned(dout, size))
    return c.bad(PLR_ERR_INVALID, "dx and dout must be aligned to their element type");
  a.x = dx;
  a.out = dout;
  a.n = n;
  a.d = d;
  a.ldx = ldx;
  a.ldo = ldo;
  rc = c.begin(device_id, hip_stream);
  if (rc != PLR_OK || n == 0) return rc;
  switch (type) {
    case PLR_F64: launch_dropout<double>(a, c.stream); break;
    case PLR_F32: launch_dropout<float>(a, c.stream); break;
    case PLR_BF16: launch_dropout<__bf16>(a, c.stream); break;
    default: launch_dropout<_Float16>(a, c.stream); break;
  }
  return c.launched();
}

int64_t plr_mxfp_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  (void)m;
  (void)n;
  (void)k;
  return 0;
}

int plr_mxfp_matmul(int device_id, void* hip_stream, int64_t m, int64_t n, int64_t k,
                    const uint8_t* da, int64_t lda, const uint8_t* dsa, int64_t ldsa,
                    const uint8_t* db, int64_t ldb, const uint8_t* dsb, int64_t ldsb, double alpha,
                    const plr_dropout* drop, void* dc, unsigned type, int64_t ldc, void* workspace,
                    int64_t workspace_bytes) {
  Call c("plr_mxfp_matmul");
  const size_t size = type_size(type);
  if (size == 0 || type == PLR_F64)
    return c.bad(PLR_ERR_INVALID, "the result is PLR_F32, PLR_BF16 or PLR_F16");
  if (m < 0 || n < 0 || k < 1) return c.bad(PLR_ERR_INVALID, "need m >= 0, n >= 0 and k >= 1");
  if (m > (int64_t)1 << 31 || n > (int64_t)1 << 31)
    return c.bad(PLR_ERR_INVALID, "m and n must be at most 2^31");
  const int64_t most = (int64_t)1 << 23;
  if (k > 2 * most || lda > most || ldb > most || ldsa > most || ldsb > most)
    return c.bad(PLR_ERR_INVALID, "k must be at most 2^24 and a pitch of codes or scales 2^23 bytes");
  if (lda % 64 != 0 || ldb % 64 != 0 || lda < plr_mxfp_code_pitch(k) || ldb < plr_mxfp_code_pitch(k))
    return c.bad(PLR_ERR_INVALID, "code pitches must be multiples of 64 and at least plr_mxfp_code_pitch(k)");
  if (ldsa % 4 != 0 || ldsb % 4 != 0 || ldsa < plr_mxfp_scale_pitch(k) || ldsb < plr_mxfp_scale_pitch(k))
    return c.bad(PLR_ERR_INVALID, "scale pitches must be multiples of 4 and at least plr_mxfp_scale_pitch(k)");
  if (ldc < n) return c.bad(PLR_ERR_INVALID, "ldc must be >= n");
  if (!fits(m, lda, 1) || !fits(n, ldb, 1) || !fits(m, ldsa, 1) || !fits(n, ldsb, 1) || !fits(m, ldc, size))
    return c.bad(PLR_ERR_INVALID, "matrix too large to address");
  MatmulArgs a;
  double scale;
  int rc = check_mask(c, drop, &a.mask, &scale);
  if (rc != PLR_OK) return rc;
  // One factor for alpha and the mask, rounded to 32 bits once (2^-24): two multiplications could pass
  // through a number too small for 32 bits on the way to one that is not.
  const double factor = alpha * scale;
  if (alpha != 0. && isfinite(alpha) && !(fabs(factor) >= FLT_MIN && fabs(factor) <= FLT_MAX))
    return c.bad(PLR_ERR_INVALID, "alpha times the mask's factor must be 0 or a normal number of 32 bits");
  if (workspace_bytes < plr_mxfp_matmul_workspace(m, n, k))
    return c.bad(PLR_ERR_INVALID, "workspace smaller than plr_mxfp_matmul_workspace(m, n, k)");
  (void)workspace;  // none of the kernels asks for any
  if (m > 0 && n > 0) {
    if (!da || !dsa || !db || !dsb || !dc)
      return c.bad(PLR_ERR_INVALID, "device pointers must not be NULL");
    if (!aligned(da, 16) || !aligned(db, 16)) return c.bad(PLR_ERR_INVALID, "da and db must be 16-byte aligned");
    if (!aligned(dsa, 4) || !aligned(dsb, 4)) return c.bad(PLR_ERR_INVALID, "dsa and dsb must be 4-byte aligned");
    if (!aligned(dc, size)) return c.bad(PLR_ERR_INVALID, "dc must be aligned to its element type");
  }
  a.a = da;
  a.b = db;
  a.sa = dsa;
  a.sb = dsb;
  a.lda = lda;
  a.ldb = ldb;
  a.ldsa = ldsa;
  a.ldsb = ldsb;
  a.m = m;
  a.n = n;
  a.chunks = (int)ceil_div(k, 128);
  a.c = dc;
  a.ldc = ldc;
  a.factor = (float)factor;
  a.row0 = a.col0 = 0;
  rc = c.begin(device_id, hip_stream);
  if (rc != PLR_OK || m == 0 || n == 0) return rc;
  const bool dr = drop != nullptr && a.mask.threshold > 0;
  if (!launch_matmul(a, type == PLR_F32 ? 0 : type == PLR_BF16 ? 1 : 2, dr, c.cus, c.stream))
    return c.bad(PLR_ERR_INVALID, "matrix too large for one launch");
  return c.launched();
}

}  // extern "C"

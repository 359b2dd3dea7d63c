// C[i, j] = alpha * sum over k of A[i, k] B[j, k], A and B in microscaled 4-bit floating point
// with their blocks along k, sums in 32 bits on the scaled matrix instruction.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "plr_mxfp.hpp"

namespace plr_mx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct MatmulArgs {
  const uint8_t *a, *b, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;
  int64_t m, n;
  int chunks;  // of 128 values along k
  void* c;
  int64_t ldc;
  float factor;  // alpha times what the mask multiplies kept values by
  int64_t row0, col0;  // where c's first element stands in the matrix that the mask belongs to
  Mask mask;
};

// One block of 32 values, in the low half of the instruction's operand.
__device__ __forceinline__ v8i operand(v4i w) {
  return __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
}

template <int SEL>
__device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(a), operand(b), c, 4, 4, SEL, sa,
                                                          SEL, sb);
}

// ------------------------------------------------------------------- epilogue
template <typename T>
struct Out8 {
  T v[8];
};
// 16 bytes at a time on any alignment (the device's global stores need none)
typedef int v4w __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void store_whole(T* c, const Out8<T>& o) {
  struct Words {
    v4w w[sizeof(T) / 2];
  };
  const Words w = __builtin_bit_cast(Words, o);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<v4w*>(c)[i] = w.w[i];
}

// Columns j .. j + 7 of row i (j a multiple of 8): factor, dropout, one rounding.
template <typename T, bool DROP>
__device__ __forceinline__ Out8<T> finish8(const MatmulArgs& p, int64_t i, int64_t j, v4f lo, v4f hi) {
  const unsigned drops = DROP ? drop_marks(p.mask, i + p.row0, (unsigned)((j + p.col0) >> 3)) : 0u;
  Out8<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = p.factor * (e < 4 ? lo[e & 3] : hi[e & 3]);
    if (DROP && (drops >> 4 * e & 1)) v = 0.f;
    o.v[e] = (T)v;
  }
  return o;
}

// A wave's 16 x (16 FN) piece of C, rows i0 .., columns j0 ..; lane (r16, q) holds columns
// 32 (y / 2) + 8 q .. + 7 of row r16 in acc[y], acc[y + 1] (y even).  Tiles that lie inside C are
// stored as they are held; those at its edge go through 1 KB of LDS per
// wave and 32 columns, so that the code with the comparisons is there once and not for every register.
template <typename T, bool DROP, int FN>
__device__ __forceinline__ void store_piece(const MatmulArgs& p, int64_t i0, int64_t j0, const v4f* acc, int r16,
                                            int q) {
  T* c = static_cast<T*>(p.c) + (i0 + r16) * p.ldc + j0 + q * 8;
#pragma unroll
  for (int y = 0; y < FN; y += 2)
    store_whole(c + y * 16, finish8<T, DROP>(p, i0 + r16, j0 + y * 16 + q * 8, acc[y], acc[y + 1]));
}
template <typename T, bool DROP, int FN>
__device__ __forceinline__ void store_edge_piece(const MatmulArgs& p, int64_t i0, int64_t j0, const v4f* acc,
                                                 int r16, int q, v4f* lds) {
  // lds: FN / 2 x 64 lanes x 2
#pragma unroll
  for (int y = 0; y < FN; ++y) lds[((y >> 1) * 64 + q * 16 + r16) * 2 + (y & 1)] = acc[y];
  const int64_t i = i0 + r16;
#pragma unroll 1
  for (int y = 0; y < FN / 2; ++y) {
    const int64_t j = j0 + y * 32 + q * 8;
    if (i >= p.m || j >= p.n) continue;
    const v4f* from = lds + (y * 64 + q * 16 + r16) * 2;
    const Out8<T> o = finish8<T, DROP>(p, i, j, from[0], from[1]);
    T* c = static_cast<T*>(p.c) + i * p.ldc + j;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e < p.n) c[e] = o.v[e];
  }
}

// Workgroups that follow each other go to the 8 XCDs in turn: give every XCD a run of tiles, and
// lay a run out in groups of 8 tile rows, so that the tiles an XCD works on at a time share their
// rows of A and B in its L2.
__device__ __forceinline__ void tile_of(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned& tm,
                                        unsigned& tn) {
  const unsigned total = tiles_m * tiles_n, per = total / 8, rem = total % 8;
  const unsigned xcd = id % 8;
  const unsigned t = xcd * per + min(xcd, rem) + id / 8;
  const unsigned group = t / (8 * tiles_n), first = group * 8;
  const unsigned height = min(8u, tiles_m - first), in = t - group * 8 * tiles_n;
  tm = first + in % height;
  tn = in / height;
}

// ------------------------------------------------------------------- large products
// A workgroup owns BM x BN of C, a wave WM x WN, in 16 x 16 x 128 instructions: lane l holds block
// l / 16 (32 values, 16 bytes, one scale byte) of row l % 16.  The rows of B go in as the
// instruction's first operand, so that a lane's four sums are four columns of one row of C, and a
// pair of 16-row pieces is dealt out so that they are eight: 16 consecutive bytes of bfloat16.
//
// 128 values of k are a step.  Codes pass through a ring of four stages in LDS, filled by
// asynchronous loads three steps ahead; a step's pieces of B and its first two of A were read
// from LDS during the step before, the other pieces of A two ahead of their use.  Within a row's
// 64 bytes of a stage the four blocks are permuted by the row number, so that the 16 rows a wave
// reads at once lie on different banks.
//
// 8192^3 in 271 to 280 us, 3.9 to 4.1 PFLOP/s; bound by power (the clock falls to 1.6 GHz) and by LDS: a step takes
// 1500 cycles, the matrix instructions of its two waves per SIMD 1024.
//
// Scales go the same way, 16 bytes per row and group of four steps, in a ring of three groups; a
// lane picks its block's four bytes into one word once per group, and the instruction selects the
// byte of its step.
// The asynchronous loads are written as instructions: the compiler holds every later read of LDS
// until all of them have landed, whichever stage it reads.  They have no register results; the
// waits are the step's own.
__device__ __forceinline__ void copy_to_lds(const uint8_t* base, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

__device__ __forceinline__ void copy_word_to_lds(const uint8_t* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               ::"s"(lds), "v"(src) : "memory", "m0");
}

template <typename T, bool DROP, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void matmul_tiles(MatmulArgs p, unsigned tiles_m,
                                                                              unsigned tiles_n) {
  constexpr int NT = 64 * (BM / WM) * (BN / WN);
  constexpr int FM = WM / 16, FN = WN / 16;        // 16-row pieces of a wave
  constexpr int LA = BM * 4 / NT, LB = BN * 4 / NT;  // asynchronous loads per thread and step
  constexpr int ROWS = BM + BN;
  // a group's scales: a quarter of the rows per step, 16 rows of four words to a wave's load; waves
  // that are over repeat the first ones'
  constexpr int UNITS = ROWS / 64;
  static_assert(UNITS <= NT / 64 && ROWS % 64 == 0, "one load of scales per thread and step");
  static_assert(LA + LB <= FM && FN <= FM && FM >= 4, "a step's loads and reads fit its rows of instructions");
  __shared__ v4i stage[4][ROWS * 4];
  __shared__ v4i scale[3][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const int kc = p.chunks;

  // what this thread loads: row tid / 4 (+ NT / 4 * i) of the tile, block (tid % 4) ^ (row's permutation)
  const int lr = tid >> 2;
  const int ka = (tid & 3) ^ ((lr >> 1) & 3), kb = (tid & 3) ^ (((lr >> 1) & 1) | ((lr >> 2) & 2));
  const uint8_t* const abase = p.a + m0 * p.lda;
  const uint8_t* const bbase = p.b + n0 * p.ldb;
  unsigned aoff[LA], boff[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i)
    aoff[i] = (unsigned)(min((int64_t)(lr + NT / 4 * i), p.m - 1 - m0) * p.lda + ka * 16);
#pragma unroll
  for (int i = 0; i < LB; ++i)
    boff[i] = (unsigned)(min((int64_t)(lr + NT / 4 * i), p.n - 1 - n0) * p.ldb + kb * 16);
  const unsigned lds0 = lds_address(&stage[0][0]) + (unsigned)wave * 1024u;
  // load i of the LA + LB that bring step k's codes into stage st
  auto fill = [&](int st, int k, int i) {
    const int64_t at = (int64_t)min(k, kc - 1) * 64;
    const unsigned to = lds0 + (unsigned)(st * ROWS * 64 + i * NT * 16);
    if (i < LA) copy_to_lds(abase + at, aoff[i], to);
    else copy_to_lds(bbase + at, boff[i - LA], to);
  };
  // load i brings the words of steps k .. k + 3 (the last step's again behind the end) of a quarter
  // of the rows into ring place `to`
  const int unit = wave < UNITS ? wave : wave - UNITS;
  const uint8_t* srow[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ROWS / 4 * i + unit * 16 + (lane >> 2);
    srow[i] = r < BM ? p.sa + min(m0 + r, p.m - 1) * p.ldsa : p.sb + min(n0 + r - BM, p.n - 1) * p.ldsb;
  }
  const unsigned lds1 = lds_address(&scale[0][0]) + (unsigned)unit * 256u;
  auto fill_scales = [&](int to, int k, int i) {
    copy_word_to_lds(srow[i] + (int64_t)min(k + (lane & 3), kc - 1) * 4,
                     lds1 + (unsigned)(to * ROWS * 16 + i * ROWS * 4));
  };

  // rows of the pieces: A straight, B dealt out by eights
  const int arow = wm + r16;
  const int brow = wn + (r16 >> 2) * 8 + (r16 & 3);
  const int apos = arow * 4 + (q ^ ((arow >> 1) & 3));  // + 64 per piece: 16 rows on, same permutation
  auto bpos = [&](int f) {
    const int r = brow + (f >> 1) * 32 + (f & 1) * 4;
    return (BM + r) * 4 + (q ^ (((r >> 1) & 1) | ((r >> 2) & 2)));
  };
  auto read_a = [&](int st, int f) { return stage[st][apos + 64 * f]; };
  auto read_b = [&](int st, int f) { return stage[st][bpos(f)]; };
  // bytes q of a row's four words, in one word
  const unsigned pick0 = 0x0c0c0400u + 0x0101u * q, pick1 = 0x04000c0cu + 0x01010000u * q;
  auto scales_of = [&](int from, int row) {
    const v4i w = scale[from][row];
    return (int)(__builtin_amdgcn_perm(w[1], w[0], pick0) | __builtin_amdgcn_perm(w[3], w[2], pick1));
  };
  auto scale_a = [&](int from, int f) { return scales_of(from, arow + 16 * f); };
  auto scale_b = [&](int from, int f) { return scales_of(from, BM + brow + (f >> 1) * 32 + (f & 1) * 4); };
  v4i fa[FM], fb[FN], na[2], nb[FN];  // pieces of this step and of the next
  int xa[FM], xb[FN], ya[FM], yb[FN];
  v4f acc[FM][FN];
#pragma unroll
  for (int x = 0; x < FM; ++x)
#pragma unroll
    for (int y = 0; y < FN; ++y) acc[x][y] = v4f{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    fill_scales(0, 0, i);
    fill_scales(1, 4, i);
  }
#pragma unroll
  for (int st = 0; st < 3; ++st)
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) fill(st, st, i);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LA + LB) : "memory");
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    fb[f] = read_b(0, f);
    xb[f] = scale_b(0, f);
  }
#pragma unroll
  for (int f = 0; f < FM; ++f) xa[f] = scale_a(0, f);
  fa[0] = read_a(0, 0);
  fa[1] = read_a(0, 1);

  // Step J of a group of four, k the group's first.  The codes of step k + J + 1 have arrived when
  // at most the loads of the step after it are under way; those of step k + J + 3 leave for the
  // stage that step k + J - 1 was read from, and a quarter of the scales of two groups on.  The
  // next group's scales are read in step 3.
#define PLR_STEP(J)                                                                              \
  {                                                                                              \
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LA + LB + 1) : "memory");                           \
    __builtin_amdgcn_s_barrier();                                                                \
    __builtin_amdgcn_sched_barrier(0);                                                           \
    _Pragma("unroll") for (int x = 0; x < FM; ++x) {                                             \
      if (x + 2 < FM) fa[x + 2] = read_a(J, x + 2);                                              \
      if (x < LA + LB) fill((J + 3) & 3, k + J + 3, x);                                          \
      if (x == FM - 1) fill_scales(place == 0 ? 2 : place - 1, k + 8, J);                        \
      if (x >= FM - FN) nb[x - (FM - FN)] = read_b((J + 1) & 3, x - (FM - FN));                  \
      if (x >= FM - 2) na[x - (FM - 2)] = read_a((J + 1) & 3, x - (FM - 2));                     \
      if (J == 3) {                                                                              \
        ya[x] = scale_a(place == 2 ? 0 : place + 1, x);                                          \
        if (x < FN) yb[x] = scale_b(place == 2 ? 0 : place + 1, x);                              \
      }                                                                                          \
      _Pragma("unroll") for (int y = 0; y < FN; ++y) acc[x][y] =                                 \
          mfma<J>(fb[y], fa[x], acc[x][y], xb[y], xa[x]);                                        \
      __builtin_amdgcn_sched_barrier(0);                                                         \
    }                                                                                            \
    _Pragma("unroll") for (int f = 0; f < FN; ++f) fb[f] = nb[f];                                \
    fa[0] = na[0];                                                                               \
    fa[1] = na[1];                                                                               \
    if (J == 3) {                                                                                \
      _Pragma("unroll") for (int f = 0; f < FM; ++f) xa[f] = ya[f];                              \
      _Pragma("unroll") for (int f = 0; f < FN; ++f) xb[f] = yb[f];                              \
      place = place == 2 ? 0 : place + 1;                                                        \
    }                                                                                            \
  }
  int k = 0, place = 0;  // place: of the group's scales in the ring
  for (; k + 4 <= kc; k += 4) {
    PLR_STEP(0)
    PLR_STEP(1)
    PLR_STEP(2)
    PLR_STEP(3)
  }
  if (k < kc) PLR_STEP(0)
  if (k + 1 < kc) PLR_STEP(1)
  if (k + 2 < kc) PLR_STEP(2)
#undef PLR_STEP
  // the loads of the steps behind the last one still write to LDS
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (m0 + BM <= p.m && n0 + BN <= p.n) {
#pragma unroll
    for (int x = 0; x < FM; ++x)
      store_piece<T, DROP, FN>(p, m0 + wm + 16 * x, n0 + wn, acc[x], r16, q);
  } else {
    __builtin_amdgcn_s_barrier();  // every wave's loads have landed
    v4f* const mine = reinterpret_cast<v4f*>(&stage[0][0]) + wave * (FN / 2 * 128);
#pragma unroll
    for (int x = 0; x < FM; ++x)
      store_edge_piece<T, DROP, FN>(p, m0 + wm + 16 * x, n0 + wn, acc[x], r16, q, mine);
  }
}

// ------------------------------------------------------------------- few rows on one side
// A few rows of the one operand ("few") against many of the other: bound by the bytes of the many,
// which are read once, straight into the instruction's operands (1 x 16384 x 8192: 14 us,
// 5.1 TB/s).  A workgroup owns 16 FX rows of the many and 16 FY of the few; its W waves divide k, and
// their sums meet in LDS in wave order.  Codes of four chunks are requested at once: 256 consecutive bytes of a row.  The same, in
// pieces of 64 x 32 and 32 x 32, serves small products, which have too few large tiles to fill the
// device.  Rows a power of two of bytes apart meet in the same channels of the L2 cache
// (256 x 256 x 16384: 20 us, where its bytes alone are 4): 16 waves to a piece make it slower.
struct FewArgs {
  MatmulArgs p;
  const uint8_t *x, *y, *sx, *sy;  // many, few
  int64_t ldx, ldy, ldsx, ldsy;
  int64_t rows;  // of x
  int64_t few;   // rows of y
};

struct alignas(4) Words4 {
  int w[4];
};

template <typename T, bool DROP, int FY, int FX, int W, bool SWAP>
__global__ __launch_bounds__(64 * W) void matmul_few(FewArgs a) {
  __shared__ v4f part[W > 1 ? W - 1 : 1][FX * FY][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int64_t x0 = (int64_t)blockIdx.x * (16 * FX), y0 = (int64_t)blockIdx.y * (16 * FY);
  const uint8_t *px[FX], *qx[FX], *py[FY], *qy[FY];
#pragma unroll
  for (int f = 0; f < FX; ++f) {
    const int64_t r = min(x0 + 16 * f + r16, a.rows - 1);
    px[f] = a.x + r * a.ldx + q * 16;
    qx[f] = a.sx + r * a.ldsx;
  }
#pragma unroll
  for (int f = 0; f < FY; ++f) {
    const int64_t r = min(y0 + 16 * f + r16, a.few - 1);
    py[f] = a.y + r * a.ldy + q * 16;
    qy[f] = a.sy + r * a.ldsy;
  }
  v4f acc[FX][FY];
#pragma unroll
  for (int x = 0; x < FX; ++x)
#pragma unroll
    for (int y = 0; y < FY; ++y) acc[x][y] = v4f{0.f, 0.f, 0.f, 0.f};
  // this wave's chunks: whole groups of four, shares differing by one group at most
  const int groups = (a.p.chunks + 3) / 4;
  const int k0 = (int)((int64_t)groups * wave / W) * 4;
  const int k1 = min((int)((int64_t)groups * (wave + 1) / W) * 4, a.p.chunks);
  // bytes q of a row's four scale words, in one word
  const unsigned pick0 = 0x0c0c0400u + 0x0101u * q, pick1 = 0x04000c0cu + 0x01010000u * q;
  auto scales = [&](const uint8_t* s, int k) {
    const Words4 w = *reinterpret_cast<const Words4*>(s + (int64_t)k * 4);
    return (int)(__builtin_amdgcn_perm(w.w[1], w.w[0], pick0) | __builtin_amdgcn_perm(w.w[3], w.w[2], pick1));
  };
  auto codes = [&](const uint8_t* s, int k) { return *reinterpret_cast<const v4i*>(s + (int64_t)k * 64); };
  int k = k0;
  for (; k + 4 <= k1; k += 4) {
    v4i cx[4][FX], cy[4][FY];
    int sx[FX], sy[FY];
#pragma unroll
    for (int f = 0; f < FX; ++f) sx[f] = scales(qx[f], k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int f = 0; f < FX; ++f) cx[j][f] = codes(px[f], k + j);
#pragma unroll
    for (int f = 0; f < FY; ++f) sy[f] = scales(qy[f], k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int f = 0; f < FY; ++f) cy[j][f] = codes(py[f], k + j);
#pragma unroll
    for (int x = 0; x < FX; ++x)
#pragma unroll
      for (int y = 0; y < FY; ++y) {
        acc[x][y] = mfma<0>(cx[0][x], cy[0][y], acc[x][y], sx[x], sy[y]);
        acc[x][y] = mfma<1>(cx[1][x], cy[1][y], acc[x][y], sx[x], sy[y]);
        acc[x][y] = mfma<2>(cx[2][x], cy[2][y], acc[x][y], sx[x], sy[y]);
        acc[x][y] = mfma<3>(cx[3][x], cy[3][y], acc[x][y], sx[x], sy[y]);
      }
  }
  for (; k < k1; ++k) {
#pragma unroll
    for (int x = 0; x < FX; ++x)
#pragma unroll
      for (int y = 0; y < FY; ++y)
        acc[x][y] = mfma<0>(codes(px[x], k), codes(py[y], k), acc[x][y], qx[x][(int64_t)k * 4 + q],
                            qy[y][(int64_t)k * 4 + q]);
  }
  if (W > 1) {
    if (wave > 0) {
#pragma unroll
      for (int x = 0; x < FX; ++x)
#pragma unroll
        for (int y = 0; y < FY; ++y) part[wave - 1][x * FY + y][lane] = acc[x][y];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int x = 0; x < FX; ++x)
#pragma unroll
      for (int y = 0; y < FY; ++y)
#pragma unroll
        for (int w = 0; w < W - 1; ++w) acc[x][y] += part[w][x * FY + y][lane];
  }
  // lane (r16, q): rows x0 + 16 x + 4 q .. + 3 of the many, row y0 + 16 y + r16 of the few
#pragma unroll
  for (int x = 0; x < FX; ++x)
#pragma unroll
    for (int y = 0; y < FY; ++y) {
      const int64_t xr = x0 + 16 * x + 4 * q, yr = y0 + 16 * y + r16;
      if (xr >= a.rows || yr >= a.few) continue;
      unsigned drops = 0;
      if (DROP && !SWAP)
        drops = drop_marks(a.p.mask, yr + a.p.row0, (unsigned)((xr + a.p.col0) >> 3)) >> 4 * (xr & 7);
      T out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = a.p.factor * acc[x][y][e];
        if (DROP && SWAP)
          drops = drop_marks(a.p.mask, xr + e + a.p.row0, (unsigned)((yr + a.p.col0) >> 3)) >> 4 * (yr & 7) << 4 * e;
        if (DROP && (drops >> 4 * e & 1)) v = 0.f;
        out[e] = (T)v;
      }
      T* c = static_cast<T*>(a.p.c);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (xr + e < a.rows) c[SWAP ? (xr + e) * a.p.ldc + yr : yr * a.p.ldc + xr + e] = out[e];
    }
}

// ------------------------------------------------------------------- launch
template <int BM, int BN, int WM, int WN>
inline bool launch_tiles(const MatmulArgs& a, int type, bool drop, hipStream_t st) {
  const int64_t tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
  if (tm > 0x7fffff / tn) return false;
  auto f = type == 0 ? (drop ? matmul_tiles<float, true, BM, BN, WM, WN> : matmul_tiles<float, false, BM, BN, WM, WN>)
           : type == 1 ? (drop ? matmul_tiles<__bf16, true, BM, BN, WM, WN>
                               : matmul_tiles<__bf16, false, BM, BN, WM, WN>)
                       : (drop ? matmul_tiles<_Float16, true, BM, BN, WM, WN>
                               : matmul_tiles<_Float16, false, BM, BN, WM, WN>);
  hipLaunchKernelGGL(f, dim3((unsigned)(tm * tn)), dim3(64 * (BM / WM) * (BN / WN)), 0, st, a, (unsigned)tm,
                     (unsigned)tn);
  return true;
}

template <typename T, bool DROP, int FY, int FX, int W>
inline void launch_few_as(const FewArgs& a, bool swap, hipStream_t st) {
  auto f = swap ? matmul_few<T, DROP, FY, FX, W, true> : matmul_few<T, DROP, FY, FX, W, false>;
  const dim3 grid((unsigned)((a.rows + 16 * FX - 1) / (16 * FX)), (unsigned)((a.few + 16 * FY - 1) / (16 * FY)));
  hipLaunchKernelGGL(f, grid, dim3(64 * W), 0, st, a);
}
template <typename T, bool DROP>
inline void launch_few(const FewArgs& a, bool swap, int cus, int squares, hipStream_t st) {
  if (squares == 1) return launch_few_as<T, DROP, 2, 2, 8>(a, swap, st);
  if (squares == 2) return launch_few_as<T, DROP, 4, 2, 4>(a, swap, st);
  const int64_t fy = (a.few + 15) / 16;
  const int64_t pieces = (a.rows + 15) / 16;
  if (fy == 1) {
    // few workgroups: more waves of each share k (1 x 256 x 16384 7.7 us)
    if (pieces < (int64_t)cus * 4 && a.p.chunks >= 16) launch_few_as<T, DROP, 1, 1, 8>(a, swap, st);
    else launch_few_as<T, DROP, 1, 1, 4>(a, swap, st);
  } else if (pieces >= (int64_t)cus * 2) {
    // two pieces of the many share what is loaded of the few, where that leaves a workgroup per
    // compute unit (48 x 16384 x 8192: 26 us, with one piece 38; 32 x 4096 x 4096: 6.9 and 5.7)
    if (fy == 2) launch_few_as<T, DROP, 2, 2, 4>(a, swap, st);
    else if (fy == 3) launch_few_as<T, DROP, 3, 2, 4>(a, swap, st);
    else launch_few_as<T, DROP, 4, 2, 4>(a, swap, st);
  } else {
    if (fy == 2) launch_few_as<T, DROP, 2, 1, 4>(a, swap, st);
    else if (fy == 3) launch_few_as<T, DROP, 3, 1, 4>(a, swap, st);
    else launch_few_as<T, DROP, 4, 1, 4>(a, swap, st);
  }
}
// Up to 32 rows always; up to 64 where tiles of 128 would leave half the device idle (48 x 16384 x
// 8192: tiles 25 us, this 26; 33 x 9000 x 4100: 12 and 10).
inline bool few_rows(const MatmulArgs& p, int cus) {
  const int64_t few = std::min(p.m, p.n), many = std::max(p.m, p.n);
  return few <= 32 || (few <= 64 && many < (int64_t)cus * 64);
}
constexpr int64_t kMostFewRows = (int64_t)0x7fffff * 16;
// squares: 0 for few rows on one side; 1, 2: a small product in pieces of 32 x 32 or 64 x 32.
inline bool launch_few_rows(const MatmulArgs& p, int type, bool drop, int cus, int squares, hipStream_t st) {
  const bool swap = p.n < p.m;  // few columns of C: the rows of A are the many
  FewArgs a;
  a.p = p;
  a.x = swap ? p.a : p.b;
  a.y = swap ? p.b : p.a;
  a.sx = swap ? p.sa : p.sb;
  a.sy = swap ? p.sb : p.sa;
  a.ldx = swap ? p.lda : p.ldb;
  a.ldy = swap ? p.ldb : p.lda;
  a.ldsx = swap ? p.ldsa : p.ldsb;
  a.ldsy = swap ? p.ldsb : p.ldsa;
  a.rows = swap ? p.m : p.n;
  a.few = swap ? p.n : p.m;
  if (a.rows > kMostFewRows || a.few > 65535 * 16) return false;
  auto f = type == 0 ? (drop ? launch_few<float, true> : launch_few<float, false>)
           : type == 1 ? (drop ? launch_few<__bf16, true> : launch_few<__bf16, false>)
                       : (drop ? launch_few<_Float16, true> : launch_few<_Float16, false>);
  f(a, swap, cus, squares, st);
  return true;
}

// How a product is cut up, by the microseconds each way is expected to take; constants from timing
// all of them over sizes from 256 x 256 x 16384 to 16384 x 8192 x 4096 on an idle device of 256
// compute units (a launch alone counts 5).  What is written of C counts nothing here: over a few steps
// of k into a large C the choice is not borne out by timing.  S: steps of 128 along k.
//   tiles of 256 x 256, one to a compute unit at a time    12 + 0.89 S a round   (8192^3: 271 us)
//   tiles of 128 x 256                                     7.6 + 0.57 S a round  (8192^3: 351)
//   tiles of 128 x 128, two to a compute unit              3.4 + 0.74 S a round  (8192^3: 397)
//                       no more than compute units         3 + 0.27 S
//   64 x 32 and 32 x 32 pieces straight from memory: what they load over and over, or one wave's
//   share of k                          (512 x 512 x 8192: 16 and 12 us, tiles of 128 x 128 19)
enum Cut { kTiles256, kTiles128x256, kTiles128, kPieces64, kPieces32 };
struct Plan {
  Cut cut;
  double us;
};
inline Plan plan_matmul(int64_t m, int64_t n, int chunks, int cus) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
  auto rounds = [&](int64_t t, int64_t at_once) { return (double)((t + at_once - 1) / at_once); };
  const double s = chunks, work = (double)m * (double)n * 128. * s;
  const int64_t small = tiles(128, 128);
  const Plan ways[] = {
      {kTiles256, 5 + rounds(tiles(256, 256), cus) * (12 + 0.89 * s)},
      {kTiles128x256, 5 + rounds(tiles(128, 256), cus) * (7.6 + 0.57 * s)},
      {kTiles128, small <= cus ? 8 + 0.27 * s : 6 + rounds(small, 2 * cus) * (3.4 + 0.74 * s)},
      {kPieces64, 5 + std::max(3.6e-9 * work, 0.22 * s)},
      {kPieces32, 5 + std::max(5e-9 * work, 0.13 * s)}};
  Plan best = ways[0];
  for (const Plan& w : ways)
    if (w.us < best.us && (w.cut <= kTiles128 || std::max(m, n) <= kMostFewRows)) best = w;
  return best;
}

// type: 0 float, 1 bfloat16, 2 half.  False when the grid would not fit one launch.
inline bool launch_matmul(const MatmulArgs& a, int type, bool drop, int cus, hipStream_t st) {
  if (few_rows(a, cus) && std::max(a.m, a.n) <= kMostFewRows) return launch_few_rows(a, type, drop, cus, 0, st);
  const Plan whole = plan_matmul(a.m, a.n, a.chunks, cus);
  // A few rows or columns over a multiple of 256 can cost a round of tiles of their own: they go to
  // the kernel for few rows, in a launch of theirs (4096 x 4100 x 2048: 37 us whole, 29 cut).
  const int64_t over_m = a.m % 256 <= 64 ? a.m % 256 : 0, over_n = a.n % 256 <= 64 ? a.n % 256 : 0;
  if (whole.cut <= kTiles128 && (over_m || over_n) && a.m > 256 && a.n > 256 &&
      std::max(a.m, a.n) <= kMostFewRows) {
    const double cost = plan_matmul(a.m - over_m, a.n - over_n, a.chunks, cus).us +
                        (over_m ? 7 : 0) + (over_n ? 7 : 0);
    if (cost < whole.us) {
      const int64_t size = type == 0 ? 4 : 2;
      MatmulArgs in = a;
      in.m -= over_m;
      in.n -= over_n;
      if (!launch_matmul(in, type, drop, cus, st)) return false;
      if (over_n) {  // columns at the right, all rows
        MatmulArgs r = a;
        r.n = over_n;
        r.b += in.n * a.ldb;
        r.sb += in.n * a.ldsb;
        r.c = static_cast<char*>(a.c) + in.n * size;
        r.col0 += in.n;
        if (!launch_few_rows(r, type, drop, cus, 0, st)) return false;
      }
      if (over_m) {  // rows at the bottom, the columns that are left
        MatmulArgs r = a;
        r.m = over_m;
        r.n = in.n;
        r.a += in.m * a.lda;
        r.sa += in.m * a.ldsa;
        r.c = static_cast<char*>(a.c) + in.m * a.ldc * size;
        r.row0 += in.m;
        if (!launch_few_rows(r, type, drop, cus, 0, st)) return false;
      }
      return true;
    }
  }
  switch (whole.cut) {
    case kTiles256: return launch_tiles<256, 256, 128, 64>(a, type, drop, st);
    case kTiles128x256: return launch_tiles<128, 256, 64, 64>(a, type, drop, st);
    case kTiles128: return launch_tiles<128, 128, 64, 64>(a, type, drop, st);
    case kPieces64: return launch_few_rows(a, type, drop, cus, 2, st);
    default: return launch_few_rows(a, type, drop, cus, 1, st);
  }
}

}  // namespace plr_mx

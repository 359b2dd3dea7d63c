// The pass over a shard held in microscaled 4-bit floating point (plr_pack_data): the dot
// products, sigmoid, residual, loss and gradient of plr_kernels.hpp's passes on 17/32 of a byte
// per value instead of 8, optionally with dropout of the values, arithmetic in 64 bits.
//
// Bound by instructions, not bytes: a value costs two multiply-adds in 64 bits and 1.5
// conversions for each of them, with dropout also an eighth of a generator call.  200000 x 1000: 62 to
// 65 us, of which the 6.9 instructions a value that are issued take 39; with dropout 102 to 113 and 80
// (14.4).
//
// A thread owns one block of 32 columns: its gradient sums stay in registers for the kernel's
// lifetime, theta is in LDS, a row's 32 values are 16 bytes.  A workgroup lays G = threads /
// blocks consecutive rows side by side (slots) and takes SR such row sets to a tile:
//   1. every thread forms its partial dot products of the tile, R row sets at a time, and leaves
//      them in LDS (with dropout also a bit per value that says what was kept),
//   2. the partials are summed per row in a fixed order and the row terms are evaluated, once per
//      row; the residuals go to LDS,
//   3. every thread reads the tile's codes again -- from the caches, a tile is 64 KB -- and adds
//      them to its gradient sums.
// Two barriers per tile.  The row terms are a chain of some 250 dependent instructions; with
// short tiles (the codes kept in registers from 1 to 3) the workgroup spent half its time there.
// No atomics: results are reproducible bit for bit.
//
// Wide rows go in column pieces and two launches: 1 (kPassDot), packed_residual for 2, 3
// (kPassAxpy).  12000 x 16385: 35 + 5 + 38 us.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "plr_kernels.hpp"
#include "plr_mxfp.hpp"

namespace plr {

struct PackedArgs {
  const uint8_t* codes;   // n x (16 * row_blocks) bytes
  const uint8_t* scales;  // n x row_blocks bytes
  const double* y;
  const double* theta;    // zero behind the stored columns, to whole blocks
  const double* theta_bias;
  double* part_g;         // [grid][pitch]
  double* part_loss;      // [grid]
  double* part_res;       // [grid] or nullptr
  double* h_out;          // n or nullptr
  double* z_buf;          // kPassDot: [pieces][n], each piece's part of the dot products
  unsigned* marks;        // two sweeps with dropout: what the first one dropped, a word per block
  const double* res_in;   // kPassAxpy: n
  int64_t n;
  int64_t row_blocks;     // blocks of a stored row
  int64_t pitch;          // doubles per row of part_g
  int64_t cols;           // of the stored row
  int piece;              // most blocks a workgroup takes; blockIdx.y counts pieces from the row's end
  int most_slots;         // most rows side by side
  unsigned loss_mode;
  int identity_link;
  double kept;            // dropout: the factor of what is kept
  plr_mx::Mask mask;
};

// R rows' codes of a thread's block, and their scale bytes in one word.
template <int R>
struct PackedTile {
  uint4 codes[R];
  unsigned scales;
  static_assert(R <= 4, "a byte per row");
};

// The same while its loads are under way (nothing may be computed from them yet).
template <int R>
struct PackedLoads {
  uint4 codes[R];
  unsigned char scales[R];
  double res[R];      // kPassAxpy
  unsigned marks[R];  // kPassAxpy with dropout
};
template <int R>
__device__ __forceinline__ PackedTile<R> arrived(const PackedLoads<R>& l) {
  PackedTile<R> t;
  t.scales = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    t.codes[r] = l.codes[r];
    t.scales |= (unsigned)l.scales[r] << (8 * r);
  }
  return t;
}

// Values 8 q + 2 p and 8 q + 2 p + 1 of row r, unscaled.
template <int R>
__device__ __forceinline__ plr_mx::v2f tile_values(const PackedTile<R>& t, int q, int p, int r) {
  const unsigned w = q == 0   ? t.codes[r].x
                     : q == 1 ? t.codes[r].y
                     : q == 2 ? t.codes[r].z
                              : t.codes[r].w;
  return p == 0   ? plr_mx::decode2<0>(w)
         : p == 1 ? plr_mx::decode2<1>(w)
         : p == 2 ? plr_mx::decode2<2>(w)
                  : plr_mx::decode2<3>(w);
}

// 2^(s - 127) of row r; a block that stands for NaN makes its row's dot product NaN.
template <int R>
__device__ __forceinline__ double tile_scale(const PackedTile<R>& t, int r) {
  const unsigned s = t.scales >> (8 * r) & 255u;
  return s == 255u ? __builtin_nan("") : plr_mx::scale_value_f64(s);
}

constexpr int kPackedR = 4;
// Columns of a block whose sums meet in LDS at a time: all, where a workgroup's fit.
constexpr int packed_end_columns(int threads) { return threads <= 512 ? 32 : 8; }

// The marks (bit q + 4 i: column 8 q + i) of a block's columns from `left` on.
__device__ __forceinline__ unsigned columns_behind(int64_t left) {
  unsigned m = 0;
  for (int c = 0; c < 32; ++c)
    if (c >= left) m |= 1u << ((c >> 3) + 4 * (c & 7));
  return m;
}

// STRIDE: entries between theta's column pairs in LDS, at least `blocks` (fixed, so that a thread's
// reads share one address).
template <bool GRAD, bool DROP, int MODE, int STRIDE, int SR, int NT, int MINW>
__global__ __launch_bounds__(NT, MINW) void packed_pass(PackedArgs a) {
  constexpr int R = kPackedR;
  static_assert(SR % R == 0, "whole groups of row sets");
  extern __shared__ double sm[];
  const int tid = threadIdx.x;
  const int piece = (int)(gridDim.y - 1 - blockIdx.y);  // a narrow last one is not left to the end
  const int blk0 = piece * a.piece;
  const int blocks = min(a.piece, (int)a.row_blocks - blk0);
  const int slots = min(NT / blocks, a.most_slots);
  const int max_rows = slots * SR;   // rows of a tile
  const int zpitch = blocks | 1;     // odd: a row's partials start on another bank than the next one's
  v2d* const thl = reinterpret_cast<v2d*>(sm);  // [16][STRIDE]: columns 2i, 2i + 1
  double* const zl = sm + 32 * STRIDE;          // [max_rows][zpitch]
  double* const rl = zl + (size_t)max_rows * zpitch;  // [max_rows]
  unsigned* const ml = reinterpret_cast<unsigned*>(rl + max_rows);  // [SR][NT]: dropped values
  const int slot = tid / blocks, blk = tid - slot * blocks;
  const bool active = slot < slots;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  // a lane sums up to 32 of a row's partials: the fewer waves evaluate row terms the better
  int per = 1;
  while (per < kWave && per * 32 < blocks) per *= 2;
  double acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.;
  plr_mx::MaskGroup group[4];
  if (DROP && MODE != kPassAxpy) {
#pragma unroll
    for (int q = 0; q < 4; ++q) group[q] = plr_mx::mask_group(a.mask, (unsigned)((blk0 + blk) * 4 + q));
  }
  RowSums sums;
  const double bias = a.theta_bias ? *a.theta_bias : 0.;

  // R row sets from set `set` on (behind the last row lie readable zeros: they count nothing).
  const unsigned at_lane = (unsigned)((active ? slot : 0) * a.row_blocks + blk0 + blk);
  auto load = [&](int64_t set, PackedLoads<R>& t) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t at = (set + r) * slots * a.row_blocks;  // the same for all threads
      t.codes[r] = reinterpret_cast<const uint4*>(a.codes + at * 16)[at_lane];
      t.scales[r] = (a.scales + at)[at_lane];
      if (MODE == kPassAxpy && DROP) t.marks[r] = (a.marks + at)[at_lane];
      if (MODE == kPassAxpy) t.res[r] = a.res_in[min((set + r) * slots + slot, a.n - 1)];
    }
  };
  // A block that stands for NaN and is dropped whole is 0 all the same.
  const unsigned behind = DROP ? columns_behind(a.cols - (int64_t)(blk0 + blk) * 32) : 0u;
  auto nothing_kept = [&](PackedTile<R>& t, int r, unsigned marks) {
    t.scales &= (marks | behind) == ~0u ? ~(255u << 8 * r) : ~0u;
  };
  // Zero what is dropped; marks[r]: bit q + 4 i is value 8 q + i of row r, 1 where dropped.
  auto drop = [&](int64_t set, PackedTile<R>& t, unsigned (&marks)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const plr_mx::MaskRow mr = plr_mx::mask_row(a.mask, (set + r) * slots + slot);
      const unsigned m0 = plr_mx::drop_marks(a.mask, group[0], mr);
      const unsigned m1 = plr_mx::drop_marks(a.mask, group[1], mr);
      const unsigned m2 = plr_mx::drop_marks(a.mask, group[2], mr);
      const unsigned m3 = plr_mx::drop_marks(a.mask, group[3], mr);
      t.codes[r].x &= plr_mx::kept_nibbles(m0);
      t.codes[r].y &= plr_mx::kept_nibbles(m1);
      t.codes[r].z &= plr_mx::kept_nibbles(m2);
      t.codes[r].w &= plr_mx::kept_nibbles(m3);
      marks[r] = m0 | m1 << 1 | m2 << 2 | m3 << 3;
      nothing_kept(t, r, marks[r]);
    }
  };
  auto drop_again = [&](PackedTile<R>& t, int r, unsigned marks) {
    t.codes[r].x &= plr_mx::kept_nibbles(marks & 0x11111111u);
    t.codes[r].y &= plr_mx::kept_nibbles(marks >> 1 & 0x11111111u);
    t.codes[r].z &= plr_mx::kept_nibbles(marks >> 2 & 0x11111111u);
    t.codes[r].w &= plr_mx::kept_nibbles(marks >> 3 & 0x11111111u);
    nothing_kept(t, r, marks);
  };
  auto update = [&](const PackedTile<R>& t, const double (&w)[R]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int r = 0; r < R; ++r)  // (eight sums apart between two additions to the same one)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const plr_mx::v2f x = tile_values<R>(t, q, p, r);
          acc[8 * q + 2 * p] = fma((double)x[0], w[r], acc[8 * q + 2 * p]);
          acc[8 * q + 2 * p + 1] = fma((double)x[1], w[r], acc[8 * q + 2 * p + 1]);
          asm volatile("" : "+v"(acc[8 * q + 2 * p]), "+v"(acc[8 * q + 2 * p + 1]));
        }
  };

  // The workgroup's share: consecutive groups of R row sets, shares differing by one at most, in
  // tiles of up to SR sets.
  const int64_t groups = (a.n + (int64_t)slots * R - 1) / ((int64_t)slots * R);
  const int64_t share = groups / gridDim.x, longer = groups - share * gridDim.x;
  const int64_t first = blockIdx.x * share + min((int64_t)blockIdx.x, longer);
  const int64_t end = (first + share + ((int64_t)blockIdx.x < longer ? 1 : 0)) * R;
  PackedLoads<R> nxt;
  if (first * R < end) load(first * R, nxt);
  if (MODE != kPassAxpy) {
    const v2d* src = reinterpret_cast<const v2d*>(a.theta + (int64_t)blk0 * 32);
    for (int e = tid; e < 16 * blocks; e += NT) thl[(e & 15) * STRIDE + (e >> 4)] = src[e];
    __syncthreads();
  }
  for (int64_t set0 = first * R; set0 < end; set0 += SR) {
    const int sets = (int)min((int64_t)SR, end - set0);
    const bool more = set0 + SR < end;
    if (MODE != kPassAxpy) {
      for (int s = 0; s < sets; s += R) {
        PackedTile<R> cur = arrived(nxt);
        if (s + R < sets) load(set0 + s + R, nxt);
        else if (GRAD) load(set0, nxt);
        else if (more) load(set0 + SR, nxt);
        if (DROP) {
          unsigned marks[R];
          drop(set0 + s, cur, marks);
          if (GRAD) {
#pragma unroll
            for (int r = 0; r < R; ++r) ml[(s + r) * NT + tid] = marks[r];
          }
          if (MODE == kPassDot && active) {
#pragma unroll
            for (int r = 0; r < R; ++r) (a.marks + (set0 + s + r) * slots * a.row_blocks)[at_lane] = marks[r];
          }
        }
        double part[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) part[r][0] = part[r][1] = 0.;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const v2d th = thl[i * STRIDE + blk];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const plr_mx::v2f x = tile_values<R>(cur, i >> 2, i & 3, r);
            part[r][0] = fma((double)x[0], th.x, part[r][0]);
            part[r][1] = fma((double)x[1], th.y, part[r][1]);
          }
          // here, and not all decoded first and summed behind the branch: that takes every register
#pragma unroll
          for (int r = 0; r < R; ++r) asm volatile("" : "+v"(part[r][0]), "+v"(part[r][1]));
        }
        if (active) {
#pragma unroll
          for (int r = 0; r < R; ++r)
            zl[((s + r) * slots + slot) * zpitch + blk] = (part[r][0] + part[r][1]) * tile_scale(cur, r);
        }
      }
      __syncthreads();
      const int rows = sets * slots;
      const int sub = tid & (per - 1);
      for (int q0 = 0; q0 < rows; q0 += NT / per) {
        const int q = q0 + tid / per;
        double z = 0.;
        if (q < rows) {
          const double* p = zl + q * zpitch;
#pragma unroll 4
          for (int b = sub; b < blocks; b += per) z += p[b];
        }
        for (int m = 1; m < per; m <<= 1) z += __shfl_xor(z, m, kWave);
        const int64_t row = set0 * slots + q;
        if (q < rows && sub == 0) {
          double res = 0.;
          if (row < a.n) {
            if (DROP) z *= a.kept;
            if (MODE == kPassDot) {
              a.z_buf[(int64_t)piece * a.n + row] = z;
            } else {
              double h, l;
              const double yv = a.y ? a.y[row] : 0.;
              row_terms(z + bias, yv, a.loss_mode, a.identity_link, h, l);
              sums.loss += l;
              res = h - yv;
              sums.res += res;
              if (a.h_out) store_h(a.h_out + row, h);
            }
          }
          if (GRAD) rl[q] = res;
        }
      }
      __syncthreads();
    }
    if (GRAD) {
#pragma unroll 1
      for (int s = 0; s < sets; s += R) {
        PackedTile<R> cur = arrived(nxt);
        double w[R];
        if (MODE == kPassAxpy) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            w[r] = nxt.res[r];
            if (DROP) drop_again(cur, r, nxt.marks[r]);
          }
        }
        if (s + R < sets) load(set0 + s + R, nxt);
        else if (more) load(set0 + SR, nxt);
        if (MODE == kPassAxpy) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int64_t row = (set0 + s + r) * slots + slot;
            w[r] = active && row < a.n ? w[r] * tile_scale(cur, r) : 0.;
          }
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (DROP) drop_again(cur, r, ml[(s + r) * NT + tid]);
            w[r] = active ? rl[(s + r) * slots + slot] * tile_scale(cur, r) : 0.;
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (DROP) w[r] *= a.kept;
        update(cur, w);
      }
    }
  }
  if (GRAD) {
    // The slots' sums, EC columns of a block at a time: `share` threads to a column, each in slot
    // order, then among themselves.  (EC + 1 doubles per thread keep a column's slots on different
    // banks.)
    constexpr int EC = packed_end_columns(NT);
    int share = 1;
    while (share < kWave && share * 2 * blocks * EC <= NT && share < slots) share *= 2;
#pragma unroll
    for (int c0 = 0; c0 < 32; c0 += EC) {
      __syncthreads();
      if (active) {
#pragma unroll
        for (int i = 0; i < EC; ++i) sm[tid * (EC + 1) + i] = acc[c0 + i];
      }
      __syncthreads();
      for (int e0 = 0; e0 < blocks * EC; e0 += NT / share) {
        const int e = e0 + tid / share, b = e / EC, i = e % EC;
        double g = 0.;
        if (b < blocks)
          for (int s = tid & (share - 1); s < slots; s += share) g += sm[(s * blocks + b) * (EC + 1) + i];
        for (int m = 1; m < share; m <<= 1) g += __shfl_xor(g, m, kWave);
        if (b < blocks && (tid & (share - 1)) == 0)
          a.part_g[(int64_t)blockIdx.x * a.pitch + (int64_t)(blk0 + b) * 32 + c0 + i] = g;
      }
    }
  }
  if (MODE == kPassFused) emit_row_sums<NT / kWave>(sums, lane, wave, a.part_loss, a.part_res);
}

// Between the two sweeps over wide rows: a row's dot product from its pieces' parts, in their
// order, and its terms.
__global__ __launch_bounds__(256) void packed_residual(const double* __restrict__ z, int pieces,
                                                       const double* __restrict__ y, double* __restrict__ res,
                                                       double* __restrict__ h_out, double* __restrict__ part_loss,
                                                       int64_t n, unsigned loss_mode, int identity_link,
                                                       const double* __restrict__ theta_bias,
                                                       double* __restrict__ part_res) {
  const double bias = theta_bias ? *theta_bias : 0.;
  RowSums sums;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    double s = 0., h, l;
    for (int p = 0; p < pieces; ++p) s += z[(int64_t)p * n + i];
    const double yv = y ? y[i] : 0.;
    row_terms(s + bias, yv, loss_mode, identity_link, h, l);
    if (res) res[i] = h - yv;
    if (h_out) store_h(h_out + i, h);
    sums.loss += l;
    sums.res += h - yv;
  }
  emit_row_sums<4>(sums, threadIdx.x & (kWave - 1), threadIdx.x / kWave, part_loss, part_res);
}

}  // namespace plr

// The pass over a shard held in microscaled 4-bit floating point (plr_pack_data): the dot
// products, sigmoid, residual, loss and gradient of plr_kernels.hpp's passes on 17/32 of a byte
// per value instead of 8, optionally with dropout of the values, arithmetic in 64 bits.
//
// A thread owns one block of 32 columns: its gradient sums stay in registers for the kernel's
// lifetime, theta in LDS (with it in registers too the compiler spills, 256 are all there are at
// two waves per SIMD), a row's 32 values are 16 bytes.  A workgroup lays G = threads / blocks
// consecutive rows side by side (slots), and R such row sets make a tile.  In step t
//   1. every thread forms its partial dot products of tile t and leaves them in LDS,
//   2. -- the step's one barrier --
//   3. one wave (another one each step) sums the partials of tile t per row, in a fixed order,
//      evaluates the row terms once per row and leaves the residuals in LDS,
//   4. meanwhile every thread adds tile t - 1 to its gradient sums: those residuals are a step
//      old, and the tile's codes are still in registers,
//   5. the loads of tile t + 2 leave, tile t + 1 has arrived.
// Dropout zeroes the codes when they arrive, so both uses meet the same values.  No atomics:
// results are reproducible bit for bit.
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
  double* z_buf;          // kPassDot: n
  const double* res_in;   // kPassAxpy: n
  int64_t n;
  int64_t row_blocks;     // blocks of a stored row
  int64_t pitch;          // doubles per row of part_g
  int blk0, blocks;       // the blocks this launch covers
  int slots;              // rows side by side: blockDim / blocks
  int lanes_per_row;      // threads that sum a row's partials (a power of two, at most 64)
  int z_accumulate;
  unsigned loss_mode;
  int identity_link;
  double kept;            // dropout: the factor of what is kept
  plr_mx::Mask mask;
};

constexpr int kPackedMaxThreads = 512;
constexpr int kPackedRows = 4;  // R

// R rows' codes of a thread's block, and their scale bytes in one word.
template <int R>
struct PackedTile {
  uint4 codes[R];
  unsigned scales;
  static_assert(R <= 4, "a byte per row");
};

// The compiler must not carry the decoded values of a tile from its first use to its second:
// 8 bytes per value instead of half a byte.
template <int R>
__device__ __forceinline__ void forget_decoded(PackedTile<R>& t) {
#pragma unroll
  for (int r = 0; r < R; ++r)
    asm volatile("" : "+v"(t.codes[r].x), "+v"(t.codes[r].y), "+v"(t.codes[r].z), "+v"(t.codes[r].w));
}

// f(i, row, values of columns 2i and 2i + 1) for the R * 32 values of a tile, unscaled.
template <int R, typename F>
__device__ __forceinline__ void each_value(const PackedTile<R>& t, F&& f) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const unsigned w = q == 0 ? t.codes[r].x : q == 1 ? t.codes[r].y : q == 2 ? t.codes[r].z : t.codes[r].w;
        const plr_mx::v2f v = p == 0   ? plr_mx::decode2<0>(w)
                              : p == 1 ? plr_mx::decode2<1>(w)
                              : p == 2 ? plr_mx::decode2<2>(w)
                                       : plr_mx::decode2<3>(w);
        f(4 * q + p, r, (double)v[0], (double)v[1]);
      }
    }
  }
}

// 2^(s - 127) of row r; a block that stands for NaN makes its row's dot product NaN.
template <int R>
__device__ __forceinline__ double tile_scale(const PackedTile<R>& t, int r) {
  const unsigned s = t.scales >> (8 * r) & 255u;
  return s == 255u ? __builtin_nan("") : plr_mx::scale_value_f64(s);
}

// STRIDE: entries between theta's column pairs in LDS, at least `blocks` (fixed, so that a thread's
// reads share one address).
template <bool GRAD, bool DROP, int MODE, int STRIDE, int R = kPackedRows>
__global__ __launch_bounds__(kPackedMaxThreads, 2) void packed_pass(PackedArgs a) {
  extern __shared__ double sm[];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int rows = a.slots * R;  // rows of a tile
  v2d* const thl = reinterpret_cast<v2d*>(sm);              // [16][STRIDE]: columns 2i, 2i + 1
  double* const zl = sm + (MODE == kPassAxpy ? 0 : 32 * STRIDE);  // [2][rows][blocks]
  double* const rl = zl + (size_t)2 * rows * a.blocks;      // [2][rows]
  const int slot = tid / a.blocks, blk = tid - slot * a.blocks;
  const bool active = slot < a.slots;
  const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int nwaves = nt / kWave;
  double acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.;
  if (MODE != kPassAxpy) {
    const v2d* src = reinterpret_cast<const v2d*>(a.theta + (int64_t)a.blk0 * 32);
    for (int e = tid; e < 16 * a.blocks; e += nt) thl[(e & 15) * STRIDE + (e >> 4)] = src[e];
    __syncthreads();
  }
  plr_mx::MaskGroup group[4];
  if (DROP) {
#pragma unroll
    for (int q = 0; q < 4; ++q) group[q] = plr_mx::mask_group(a.mask, (unsigned)((a.blk0 + blk) * 4 + q));
  }
  RowSums sums;
  const double bias = a.theta_bias ? *a.theta_bias : 0.;
  const int64_t ntiles = (a.n + rows - 1) / rows;

  // Rows behind the last one, and threads without a block, read a row that is there and count
  // nothing.
  const unsigned at_lane = (unsigned)((active ? slot : 0) * a.row_blocks + a.blk0 + blk);
  auto load = [&](int64_t tile, PackedTile<R>& t) {
    t.scales = 0;
    if ((tile + 1) * rows <= a.n) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t at = (tile * rows + r * a.slots) * a.row_blocks;  // the same for all threads
        t.codes[r] = reinterpret_cast<const uint4*>(a.codes + at * 16)[at_lane];
        t.scales |= (unsigned)(a.scales + at)[at_lane] << (8 * r);
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        int64_t row = tile * rows + r * a.slots + (active ? slot : 0);
        row = row < a.n ? row : a.n - 1;
        const int64_t at = row * a.row_blocks + a.blk0 + blk;
        t.codes[r] = *reinterpret_cast<const uint4*>(a.codes + at * 16);
        t.scales |= (unsigned)a.scales[at] << (8 * r);
      }
    }
  };
  auto drop = [&](int64_t tile, PackedTile<R>& t) {
    if (!DROP) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const plr_mx::MaskRow mr = plr_mx::mask_row(a.mask, tile * rows + r * a.slots + slot);
      t.codes[r].x &= plr_mx::keep_nibbles(a.mask, group[0], mr);
      t.codes[r].y &= plr_mx::keep_nibbles(a.mask, group[1], mr);
      t.codes[r].z &= plr_mx::keep_nibbles(a.mask, group[2], mr);
      t.codes[r].w &= plr_mx::keep_nibbles(a.mask, group[3], mr);
    }
  };
  auto dot = [&](PackedTile<R>& t, double* z) {
    double part[R];
#pragma unroll
    for (int r = 0; r < R; ++r) part[r] = 0.;
    v2d th;
    each_value<R>(t, [&](int i, int r, double x0, double x1) {
      if (r == 0) th = thl[i * STRIDE + blk];
      part[r] = fma(x0, th.x, part[r]);
      part[r] = fma(x1, th.y, part[r]);
      // here, and not all decoded first and summed behind the branch: that takes every register
      asm volatile("" : "+v"(part[r]));
    });
    if (active) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        z[(r * a.slots + slot) * a.blocks + blk] = part[r] * tile_scale(t, r);
    }
  };
  // Row sums and row terms: `per` lanes share a row, a wave takes 64 / per rows at a time, the
  // waves take turns from tile to tile.
  auto finish_rows = [&](int64_t tile, const double* z, double* res) {
    const int per = a.lanes_per_row, step = kWave / per, sub = lane & (per - 1);
    int first = wave - (int)(tile % nwaves);
    if (first < 0) first += nwaves;
    for (int q0 = first * step; q0 < rows; q0 += nwaves * step) {
      const int q = q0 + lane / per;
      double s = 0.;
      if (q < rows) {
        const double* p = z + (size_t)q * a.blocks;
#pragma unroll 4
        for (int b = sub; b < a.blocks; b += per) s += p[b];
      }
      for (int m = 1; m < per; m <<= 1) s += __shfl_xor(s, m, kWave);
      const int64_t row = tile * rows + q;
      if (q < rows && sub == 0) {
        double rv = 0.;
        if (row < a.n) {
          if (DROP) s *= a.kept;
          if (MODE == kPassDot) {
            a.z_buf[row] = a.z_accumulate ? a.z_buf[row] + s : s;
          } else {
            double h, l;
            const double yv = a.y ? a.y[row] : 0.;
            row_terms(s + bias, yv, a.loss_mode, a.identity_link, h, l);
            sums.loss += l;
            rv = h - yv;
            sums.res += rv;
            if (a.h_out) store_h(a.h_out + row, h);
          }
        }
        if (GRAD) res[q] = rv;
      }
    }
  };
  auto update = [&](PackedTile<R>& t, const double* w) {
    each_value<R>(t, [&](int i, int r, double x0, double x1) {
      acc[2 * i] = fma(x0, w[r], acc[2 * i]);
      acc[2 * i + 1] = fma(x1, w[r], acc[2 * i + 1]);
    });
  };

  const int64_t t0 = blockIdx.x, dt = gridDim.x;
  if (MODE == kPassAxpy) {
    PackedTile<R> cur, nxt;
    if (t0 < ntiles) load(t0, nxt);
    for (int64_t t = t0; t < ntiles; t += dt) {
      cur = nxt;
      if (t + dt < ntiles) load(t + dt, nxt);
      drop(t, cur);
      double w[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = t * rows + r * a.slots + slot;
        w[r] = active && row < a.n ? a.res_in[row] * tile_scale(cur, r) : 0.;
        if (DROP) w[r] *= a.kept;
      }
      update(cur, w);
    }
  } else {
    PackedTile<R> prev, cur, nxt;
    if (t0 < ntiles) load(t0, cur);
    if (t0 + dt < ntiles) load(t0 + dt, nxt);
    int par = 0;
    for (int64_t t = t0; t < ntiles + (GRAD ? dt : 0); t += dt, par ^= 1) {
      const bool live = t < ntiles;  // (with a gradient the last step only adds the last tile)
      if (live) {
        drop(t, cur);
        dot(cur, zl + (size_t)par * rows * a.blocks);
      }
      __syncthreads();
      if (live) finish_rows(t, zl + (size_t)par * rows * a.blocks, rl + par * rows);
      if (GRAD) {
        if (t >= t0 + dt) {
          forget_decoded(prev);
          const double* res = rl + (par ^ 1) * rows;
          double w[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            w[r] = active ? res[r * a.slots + slot] * tile_scale(prev, r) : 0.;
            if (DROP) w[r] *= a.kept;
          }
          update(prev, w);
        }
        prev = cur;
      }
      cur = nxt;
      if (t + 2 * dt < ntiles) load(t + 2 * dt, nxt);
    }
  }
  if (GRAD) {
    // the slots' sums, eight columns at a time, in slot order
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (active) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sm[tid * 8 + i] = acc[8 * q + i];
      }
      __syncthreads();
      for (int e = tid; e < a.blocks * 8; e += nt) {
        const int b = e >> 3, i = e & 7;
        double g = 0.;
        for (int s = 0; s < a.slots; ++s) g += sm[(s * a.blocks + b) * 8 + i];
        a.part_g[(int64_t)blockIdx.x * a.pitch + (int64_t)(a.blk0 + b) * 32 + 8 * q + i] = g;
      }
      __syncthreads();
    }
  }
  if (MODE == kPassFused) {
    // the waves' loss and residual sums, in wave order
    __shared__ double lx[kPackedMaxThreads / kWave], rx[kPackedMaxThreads / kWave];
    const double wl = wave_sum(sums.loss), wr = wave_sum(sums.res);
    if (lane == 0) {
      lx[wave] = wl;
      rx[wave] = wr;
    }
    __syncthreads();
    if (tid == 0) {
      double l = 0., r = 0.;
      for (int w = 0; w < nwaves; ++w) {
        l += lx[w];
        r += rx[w];
      }
      a.part_loss[blockIdx.x] = l;
      if (a.part_res) a.part_res[blockIdx.x] = r;
    }
  }
}

}  // namespace plr

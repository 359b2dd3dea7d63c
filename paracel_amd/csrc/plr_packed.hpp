// The pass over a shard held in microscaled 4-bit floating point (plr_pack_data): the dot
// products, sigmoid, residual, loss and gradient of plr_kernels.hpp's passes on 17/32 of a byte
// per value instead of 8, optionally with dropout of the values, arithmetic in 64 bits.
//
// A thread owns one block of 32 columns: its theta and its gradient sums stay in registers for
// the kernel's lifetime, a row's 32 values are 16 bytes.  A workgroup lays G = threads / blocks
// consecutive rows side by side (slots), and R such row sets make a tile.  A tile takes two
// barriers: every thread's partial dot products go to LDS, are summed per row in a fixed order by
// the threads of the workgroup, which evaluate the row terms, and the residuals come back through
// LDS to the threads, whose codes -- and keep bits -- are still in registers.  No atomics: results
// are reproducible bit for bit.
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

// The 32 values of a block times `t`, or added into `t` times w.
template <bool DROP, typename F>
__device__ __forceinline__ void each_value(uint4 codes, unsigned keep, F&& f) {
  const unsigned w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    plr_mx::v2f v[4] = {plr_mx::decode2<0>(w[q]), plr_mx::decode2<1>(w[q]),
                        plr_mx::decode2<2>(w[q]), plr_mx::decode2<3>(w[q])};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = v[i >> 1][i & 1];
      if (DROP && !(keep >> (8 * q + i) & 1u)) x = 0.f;
      f(8 * q + i, (double)x);
    }
  }
}

constexpr int kPackedMaxThreads = 512;
constexpr int kPackedRows = 4;  // R

template <bool GRAD, bool DROP, int MODE, int R>
__global__ __launch_bounds__(kPackedMaxThreads, 2) void packed_pass(PackedArgs a) {
  extern __shared__ double sm[];
  double* const zl = sm;                                     // [slots * R][blocks]
  double* const rl = sm + (size_t)a.slots * R * a.blocks;    // [slots * R]
  const int tid = threadIdx.x, nt = blockDim.x;
  const int slot = tid / a.blocks, blk = tid - slot * a.blocks;
  const bool active = slot < a.slots;
  const int rows = a.slots * R;  // rows of a tile
  double th[32], acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    th[i] = active && MODE != kPassAxpy ? a.theta[(int64_t)(a.blk0 + blk) * 32 + i] : 0.;
    acc[i] = 0.;
  }
  RowSums sums;
  const double bias = a.theta_bias ? *a.theta_bias : 0.;
  const int64_t ntiles = (a.n + rows - 1) / rows;
  for (int64_t tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
    const int64_t base = tile * rows;
    uint4 codes[R];
    unsigned sc[R], keep[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * a.slots + slot;
      codes[r] = uint4{0, 0, 0, 0};
      sc[r] = 127u;
      if (active && row < a.n) {
        const int64_t at = row * a.row_blocks + a.blk0 + blk;
        codes[r] = *reinterpret_cast<const uint4*>(a.codes + at * 16);
        sc[r] = a.scales[at];
      }
    }
    if (DROP) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        keep[r] = 0;
        const int64_t row = base + r * a.slots + slot;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          keep[r] |= plr_mx::keep8(a.mask, row, (unsigned)((a.blk0 + blk) * 4 + q)) << (8 * q);
      }
    }
    // 2^(s - 127); a block that stands for NaN makes its row's dot product NaN
    double s64[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      s64[r] = sc[r] == 255u ? __builtin_nan("") : plr_mx::scale_value_f64(sc[r]);
    if (MODE != kPassAxpy) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        double z = 0.;
        each_value<DROP>(codes[r], DROP ? keep[r] : 0u, [&](int i, double x) { z = fma(x, th[i], z); });
        if (active) zl[(r * a.slots + slot) * a.blocks + blk] = z * s64[r];
      }
      __syncthreads();
      const int P = a.lanes_per_row;
      const int sub = tid & (P - 1);
      for (int q0 = 0; q0 < rows; q0 += nt / P) {
        const int q = q0 + tid / P;
        double z = 0.;
        if (q < rows)
          for (int b = sub; b < a.blocks; b += P) z += zl[q * a.blocks + b];
        for (int m = 1; m < P; m <<= 1) z += __shfl_xor(z, m, kWave);
        const int64_t row = base + q;
        if (q < rows && sub == 0) {
          double res = 0.;
          if (row < a.n) {
            if (DROP) z *= a.kept;
            if (MODE == kPassDot) {
              a.z_buf[row] = a.z_accumulate ? a.z_buf[row] + z : z;
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
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = base + r * a.slots + slot;
        double w = 0.;
        if (active && row < a.n) w = MODE == kPassAxpy ? a.res_in[row] : rl[r * a.slots + slot];
        w *= DROP ? s64[r] * a.kept : s64[r];
        each_value<DROP>(codes[r], DROP ? keep[r] : 0u,
                         [&](int i, double x) { acc[i] = fma(x, w, acc[i]); });
      }
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
    // the waves' loss and residual sums, in wave order (waves beyond the workgroup's count as 0)
    __shared__ double lx[kPackedMaxThreads / kWave], rx[kPackedMaxThreads / kWave];
    const double wl = wave_sum(sums.loss), wr = wave_sum(sums.res);
    if ((tid & 63) == 0) {
      lx[tid >> 6] = wl;
      rx[tid >> 6] = wr;
    }
    __syncthreads();
    if (tid == 0) {
      double l = 0., r = 0.;
      for (int w = 0; w < nt / kWave; ++w) {
        l += lx[w];
        r += rx[w];
      }
      a.part_loss[blockIdx.x] = l;
      if (a.part_res) a.part_res[blockIdx.x] = r;
    }
  }
}

}  // namespace plr

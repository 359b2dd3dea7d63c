// C[i, j] = alpha * sum over k of A[i, k] B[j, k], A and B in microscaled 4-bit floating point
// with their blocks along k, sums in 32 bits on the scaled matrix instruction.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "plr_mxfp.hpp"

namespace plr_mx {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct MatmulArgs {
  const uint8_t *a, *b, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;
  int64_t m, n;
  int chunks;  // of 128 values along k
  void* c;
  int64_t ldc;
  float alpha;
  float kept;  // dropout: the factor of what is kept
  Mask mask;
};

// 16 bytes = one block of 32 values, in the low half of the instruction's operand.
__device__ __forceinline__ v8i operand(const uint8_t* p) {
  const int4 w = *reinterpret_cast<const int4*>(p);
  return v8i{w.x, w.y, w.z, w.w, 0, 0, 0, 0};
}

template <typename T>
__device__ __forceinline__ T narrow(float v) {
  return (T)v;
}

// Simple form: a wave owns 32 x 32 of C, four waves 64 x 64.  For the 16 x 16 x 128 instruction
// lane l holds row l % 16 and block l / 16 of the 128 values: 16 consecutive bytes of a code row
// and one scale byte.  Rows past the end are read as the last row and not stored.
template <typename T, bool DROP>
__global__ __launch_bounds__(256) void matmul_simple(MatmulArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)blockIdx.y * 64 + (wave >> 1) * 32;
  const int64_t j0 = (int64_t)blockIdx.x * 64 + (wave & 1) * 32;
  const int r16 = lane & 15, q = lane >> 4;
  const uint8_t *pa[2], *pb[2], *qa[2], *qb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t i = min(i0 + 16 * t + r16, p.m - 1), j = min(j0 + 16 * t + r16, p.n - 1);
    pa[t] = p.a + i * p.lda + q * 16;
    pb[t] = p.b + j * p.ldb + q * 16;
    qa[t] = p.sa + i * p.ldsa + q;
    qb[t] = p.sb + j * p.ldsb + q;
  }
  v4f acc[2][2] = {};
  for (int k = 0; k < p.chunks; ++k) {
    v8i a[2], b[2];
    int sa[2], sb[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      a[t] = operand(pa[t] + (int64_t)k * 64);
      b[t] = operand(pb[t] + (int64_t)k * 64);
      sa[t] = qa[t][(int64_t)k * 4];
      sb[t] = qb[t][(int64_t)k * 4];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y)
        acc[x][y] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[x], b[y], acc[x][y], 4, 4, 0,
                                                                     sa[x], 0, sb[y]);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + 16 * x + q * 4 + e, j = j0 + 16 * y + r16;
        if (i >= p.m || j >= p.n) continue;
        float v = p.alpha * acc[x][y][e];
        if (DROP) v = (drop_marks(p.mask, i, (unsigned)(j >> 3)) >> 4 * (j & 7) & 1) ? 0.f : v * p.kept;
        static_cast<T*>(p.c)[i * p.ldc + j] = narrow<T>(v);
      }
}

template <typename T>
inline void launch_simple(const MatmulArgs& a, bool drop, dim3 grid, hipStream_t st) {
  auto f = drop ? matmul_simple<T, true> : matmul_simple<T, false>;
  hipLaunchKernelGGL(f, grid, dim3(256), 0, st, a);
}

// type: 0 float, 1 bfloat16, 2 half.  False when the grid would not fit one launch.
inline bool launch_matmul(const MatmulArgs& a, int type, bool drop, int cus, hipStream_t st) {
  (void)cus;
  const int64_t gx = (a.n + 63) / 64, gy = (a.m + 63) / 64;
  if (gy > 65535 || gx > 0x7fffffff) return false;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (type == 0) launch_simple<float>(a, drop, grid, st);
  else if (type == 1) launch_simple<__bf16>(a, drop, grid, st);
  else launch_simple<_Float16>(a, drop, grid, st);
  return true;
}

}  // namespace plr_mx

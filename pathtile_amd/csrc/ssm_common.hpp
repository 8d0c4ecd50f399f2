// ssm_common.hpp — what the kernels of the selective state space block share:
// loads and stores of FP32 and BF16 activations, and the scalar functions.
// Activations are FP32 or BF16 and are computed on in FP32; an output is
// rounded to its type once, as it is stored.

#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace pt {

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

using f4v = __attribute__((ext_vector_type(4))) float;
using u4v = __attribute__((ext_vector_type(4))) uint32_t;

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)lo) |
         (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)hi) << 16;
}

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }

// Eight consecutive values, p aligned to 16 bytes.
__device__ __forceinline__ void load_vec(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const f4v q = *reinterpret_cast<const f4v*>(p + i);
    v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
  }
}
__device__ __forceinline__ void load_vec(const __bf16* p, float (&v)[8]) {
  const u4v q = *reinterpret_cast<const u4v*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[2 * j] = bf16_lo(q[j]), v[2 * j + 1] = bf16_hi(q[j]);
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4)
    *reinterpret_cast<f4v*>(p + i) = f4v{v[i], v[i + 1], v[i + 2], v[i + 3]};
}
__device__ __forceinline__ void store_vec(__bf16* p, const float (&v)[8]) {
  u4v q;
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = bf16_pair(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<u4v*>(p) = q;
}

// exp(v). The exponent is rounded once, to 2^-24 |v| of the result; a result
// below 2^-126 is 0.
__device__ __forceinline__ float exp_f32(float v) { return __builtin_amdgcn_exp2f(v * kLog2E); }
__device__ __forceinline__ float sigmoid_f32(float v) {
  return __builtin_amdgcn_rcpf(1.0f + exp_f32(-v));
}
// d/dp of p sigmoid(p), from sig = sigmoid(p)
__device__ __forceinline__ float silu_grad_f32(float p, float sig) {
  return sig * fmaf(p, 1.0f - sig, 1.0f);
}

// Sums of columns over `parts` rows in a fixed order: 32 columns by 32 ranges of
// rows a workgroup of 1024. column(i, &stride) is where column i begins, or
// null, and sets how far its rows are apart; done(i, sum) takes the result. Rows
// are read 128 bytes at a time, 32 of them at once: 5 us for 512 x 4096.
constexpr int kSumThreads = 1024, kSumCols = 32;
template <typename Column, typename Done>
__device__ __forceinline__ void sum_columns(long long first, long long parts, Column column, Done done) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  long long stride = 0;
  const float* p = column(first + c, &stride);
  float v = 0.0f;
  if (p) {
#pragma unroll 8
    for (long long i = k; i < parts; i += 32) v += p[i * stride];
  }
  sums[k][c] = v;
  __syncthreads();
  v = sums[c][k];
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor(v, m);
  if (c == 0) done(first + k, v);
}

}  // namespace pt

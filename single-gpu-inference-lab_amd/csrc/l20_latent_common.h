// Shared by the latent attention kernels (gfx950): element types, the 16x16x32 matrix product, the
// transposing LDS read and the chunk swizzles of their LDS tiles.
#ifndef L20_LATENT_COMMON_H_
#define L20_LATENT_COMMON_H_

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <stdio.h>

// Error reporting shared with the decode entry points (l20_pd_last_error).
namespace l20pd_host {
int32_t set_error(int32_t code, const char *msg);
void clear_error();
}  // namespace l20pd_host

namespace l20la {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kRope = 64;  // rotary dims of a latent row
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFp8Max = 448.0f;

// Two floats -> two elements of T in one dword, round to nearest even.
template <typename T> __device__ __forceinline__ int pack2(float a, float b);
template <> __device__ __forceinline__ int pack2<__bf16>(float a, float b) {
  return __builtin_bit_cast(int, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
template <> __device__ __forceinline__ int pack2<_Float16>(float a, float b) {
  return __builtin_bit_cast(int, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// D = A B + C of 16x16x32.  Lane l holds A[l % 16][8 (l / 16) + j], B[8 (l / 16) + j][l % 16] (j = 0..7)
// and C[4 (l / 16) + i][l % 16] (i = 0..3).
template <typename T> __device__ __forceinline__ f32x4 mfma(i32x4 a, i32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma<__bf16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma<_Float16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Transposing LDS read: in each group of 16 lanes, lane i's address is row i / 4, columns 4 (i % 4) .. + 3
// of a block of 4 rows by 16 columns of 16-bit elements; lane i receives column i of the four rows.
__device__ __forceinline__ i32x2 read_tr(const char *p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (lds_s16x4 *)(__attribute__((address_space(3))) char *)(p)));
}

__device__ __forceinline__ float max_groups(float x) {  // over the four lane groups of 16
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 16 bytes of zeros a lane: what rows that take no part are read from (a masked row's values still
// enter the product with a weight of 0, and 0 x NaN is NaN).
__device__ const i32x4 kZeroRow[128] = {};

}  // namespace l20la

#endif  // L20_LATENT_COMMON_H_

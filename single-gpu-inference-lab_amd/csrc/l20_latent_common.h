// Shared by the latent attention kernels (gfx950): element types, the 16x16x32 matrix product, the
// transposing LDS read and the chunk swizzles of their LDS tiles.
#ifndef L20_LATENT_COMMON_H_
#define L20_LATENT_COMMON_H_

#include <hip/hip_runtime.h>

#include <atomic>

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
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// D = A B + C of 32x32x16.  Lane l holds A[l % 32][8 (l / 32) + j], B[8 (l / 32) + j][l % 32] (j = 0..7) and
// C[8 (i / 4) + 4 (l / 32) + i % 4][l % 32] (i = 0..15).
template <typename T> __device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<__bf16>(i32x4 a, i32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<_Float16>(i32x4 a, i32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The same of 8-bit elements: lane i's address is row i / 2, columns 8 (i % 2) .. + 7 of a block of 8 rows by 16
// columns; lane i receives column i of the eight rows.
__device__ __forceinline__ i32x2 read_tr8(const char *p) {
  typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(__attribute__((address_space(3))) char *)(p));
}

// What the 16-byte chunks of row `row` are XORed with in an LDS tile whose rows are multiples of 256 bytes (all
// banks): sixteen rows differ, so a read of one chunk of each meets all banks; four consecutive rows differ in fours
// of chunks and rows eight apart in pairs, so 32 lanes of a transposing read meet all banks too, whether they take 64
// bytes of each of four rows or 32 of rows 0 .. 3 and 8 .. 11.  A permutation of the row's bits: linear under XOR.
__device__ __forceinline__ int spread_row(int row) { return (row & 3) << 2 | (row >> 3 & 1) << 1 | (row >> 2 & 1); }

// Reductions by the row swaps of the vector ALU (no LDS round trip): with both operands the same register a
// swap returns a lane's value and that of the lane 16 (32) away, in one order for both of them.
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
template <int W> __device__ __forceinline__ u32x2 swap_rows(float x) {
  const unsigned int b = __builtin_bit_cast(unsigned int, x);
  if constexpr (W == 16) return __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(b, b, false, false));
  else return __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(b, b, false, false));
}
// (by value: hipcc lowers __builtin_bit_cast of an ext_vector element to a load of element 0)
__device__ __forceinline__ float word_f(unsigned int w) { return __builtin_bit_cast(float, w); }
template <int W> __device__ __forceinline__ float max_swap(float x) {
  const u32x2 r = swap_rows<W>(x);
  return fmaxf(word_f(r[0]), word_f(r[1]));
}
template <int W> __device__ __forceinline__ float sum_swap(float x) {
  const u32x2 r = swap_rows<W>(x);
  return word_f(r[0]) + word_f(r[1]);
}
__device__ __forceinline__ float max_halves(float x) { return max_swap<32>(x); }  // over lanes l and l ^ 32
__device__ __forceinline__ float sum_halves(float x) { return sum_swap<32>(x); }
__device__ __forceinline__ float max_groups(float x) { return max_swap<32>(max_swap<16>(x)); }  // the four groups of 16
__device__ __forceinline__ float sum_groups(float x) { return sum_swap<32>(sum_swap<16>(x)); }

// The lane's number, made anew: where registers are short it is not kept.
__device__ __forceinline__ int lane_id() {
  int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
  asm volatile("" : "+v"(lane));
  return lane;
}
// Lane n's value (n: wave-uniform).
__device__ __forceinline__ float lane_f(float x, int n) {
  return word_f((unsigned int)__builtin_amdgcn_readlane(__builtin_bit_cast(int, x), n));
}
// Two products of the pairs of Ts in two words, added to x one after the other.
template <typename T> __device__ __forceinline__ float dot2(int a, int b, float x) {
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair u = __builtin_bit_cast(pair, a), v = __builtin_bit_cast(pair, b);
  return __builtin_fmaf((float)u[1], (float)v[1], __builtin_fmaf((float)u[0], (float)v[0], x));
}

// The largest of three (fmaxf quiets each operand first, one instruction more a value).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// 16 bytes a lane from global memory to LDS (lane l's land at dst + 16 l), asynchronously: they are there once
// the wave has waited for its loads (landed_and_barrier).  Not the builtin: with a builtin's load in flight the
// compiler waits for all loads before every transposing read, which ends the prefetch; a load into LDS has no
// result registers that could be taken for written.
__device__ __forceinline__ void load_lds(const void *src, uint32_t dst) {  // dst: wave-uniform
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(dst) : "memory");
}
__device__ __forceinline__ void load_lds(const void *base, uint32_t off, uint32_t dst) {  // base, dst: wave-uniform
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(dst) : "memory");
}
// The LDS address of a pointer into shared memory (the low half of a generic one).
__device__ __forceinline__ uint32_t lds_address(const void *p) { return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p); }

// All but the wave's last N loads have landed, in LDS too, and so for the workgroup's other waves.
template <int N> __device__ __forceinline__ void landed_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// LDS writes of the workgroup's waves are there; loads may be in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The running maximum of a softmax row moves only when a tile's exceeds it by more than this (log2 units): P is
// then at most 2^8 where it would be 1, which costs neither type precision (fp16 ends at 2^16).
constexpr float kRescale = 8.0f;

// A kernel's limit of dynamic LDS, raised once a device (each raise costs a launch a good part of a microsecond).
struct LdsLimit {
  std::atomic<uint64_t> devices{0};
  hipError_t raise(const void *kernel, int bytes) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if (devices.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) devices.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

// The compute units of the current device.
inline int device_cus() {
  static std::atomic<int> known[64];  // by device
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (dev < 64 && (cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  if (dev < 64) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// 16 bytes of zeros a lane: what rows that take no part are read from (a masked row's values still
// enter the product with a weight of 0, and 0 x NaN is NaN).
__device__ const i32x4 kZeroRow[128] = {};

}  // namespace l20la

#endif  // L20_LATENT_COMMON_H_

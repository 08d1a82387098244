// What the kernels over paged K/V share: metadata reads, the matrix products, and the reads of
// bf16 tiles in LDS.
#pragma once

#include "common.h"

namespace kvp {

// n / d for 0 <= n < 2^31 by a multiplication (the compiler's division is some 30
// instructions, most of them executed once per launch from a cold instruction cache).
// With l = ceil(log2 d) and mul = ceil(2^(31 + l) / d), n * mul / 2^(31 + l) exceeds n / d
// by less than n / 2^(31 + l) <= 1 / d for n < 2^31, so the floor is exact.
struct Divisor {
  uint32_t mul, shift;  // shift = l - 1 beyond the high word; d = 1: mul = 0
};
static Divisor divisor(uint32_t d) {
  if (d <= 1) return Divisor{0, 0};
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return Divisor{static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d), l - 1};
}
__device__ __forceinline__ int div_by(int n, const Divisor& d) {
  return d.mul ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), d.mul) >> d.shift) : n;
}

// A wave-uniform read of read-only metadata (context lengths, block tables) through the
// constant address space, so it compiles to a scalar load.  Scalar loads are counted
// apart from the vector loads of the K/V stream: waiting for a block id does not wait
// for the KV loads in flight (as a vector load's wait would, vector loads complete in
// order), and a block id loaded one block ahead is waited for only where it is used.
__device__ __forceinline__ int load_uniform(const int32_t* base, int64_t idx) {
  return ((const __attribute__((address_space(4))) int32_t*)(base))[idx];
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float mfma_f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ mfma_f32x4_t mfma16(u32x4_t a, u32x4_t b, mfma_f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: 8 bytes per lane, transposed as 16-bit elements across each
// 16-lane group (see the V^T operand in the kernel).
__device__ __forceinline__ uint2 lds_read_tr16(const uint16_t* lds_ptr) {
  const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4_t*)(lds_ptr));
  return __builtin_bit_cast(uint2, v);
}

// Max / sum of x over lanes l and l ^ 32 (v_permlane32_swap_b32 exchanges the wave halves:
// the first result holds lanes 0-31 in both halves, the second lanes 32-63).
__device__ __forceinline__ float half_swap_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// All LDS accesses of the wave are done: what they read may be overwritten.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Tile accesses are written out, each block with its own wait: the compiler cannot tell a
// tile from the one being filled and would wait for every load in flight.
__device__ __forceinline__ u32 lds_addr(const void* p) {
  return static_cast<u32>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)(p)));
}
// The 16 bytes at a[i] and at a[i] + 4096 (the tile's two 16-token halves), i = 0..3.
__device__ __forceinline__ void read_k_tile(const u32 (&a)[4], u32x4_t (&k)[8]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:4096\n\t"
      "ds_read_b128 %2, %9\n\tds_read_b128 %3, %9 offset:4096\n\t"
      "ds_read_b128 %4, %10\n\tds_read_b128 %5, %10 offset:4096\n\t"
      "ds_read_b128 %6, %11\n\tds_read_b128 %7, %11 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
      : "memory");
}
typedef u32 u32x2_t __attribute__((ext_vector_type(2)));
// Transposed 8-byte reads at a[i] (first half) and a[i] + 4096 (second half), i = 0..7.
__device__ __forceinline__ void read_v_tile(const u32 (&a)[8], u32x2_t (&lo)[8], u32x2_t (&hi)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %8, %16 offset:4096\n\t"
      "ds_read_b64_tr_b16 %1, %17\n\tds_read_b64_tr_b16 %9, %17 offset:4096\n\t"
      "ds_read_b64_tr_b16 %2, %18\n\tds_read_b64_tr_b16 %10, %18 offset:4096\n\t"
      "ds_read_b64_tr_b16 %3, %19\n\tds_read_b64_tr_b16 %11, %19 offset:4096\n\t"
      "ds_read_b64_tr_b16 %4, %20\n\tds_read_b64_tr_b16 %12, %20 offset:4096\n\t"
      "ds_read_b64_tr_b16 %5, %21\n\tds_read_b64_tr_b16 %13, %21 offset:4096\n\t"
      "ds_read_b64_tr_b16 %6, %22\n\tds_read_b64_tr_b16 %14, %22 offset:4096\n\t"
      "ds_read_b64_tr_b16 %7, %23\n\tds_read_b64_tr_b16 %15, %23 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(lo[4]), "=&v"(lo[5]), "=&v"(lo[6]),
        "=&v"(lo[7]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3]), "=&v"(hi[4]), "=&v"(hi[5]),
        "=&v"(hi[6]), "=&v"(hi[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
      : "memory");
}

}  // namespace kvp

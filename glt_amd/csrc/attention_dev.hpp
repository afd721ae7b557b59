// Device helpers shared by the attention kernels (attention.hip,
// attention_bwd.hip).
#pragma once

#include "common.hpp"

namespace glt {

constexpr int kHd = 128;          // head dimension

// Refuses what no attention training entry point serves (attention.hip).
glt_status check_attn_desc(const glt_attn_desc* d, const char* who);

typedef __attribute__((address_space(3))) void lds_void;
typedef uint32_t u32x2a __attribute__((ext_vector_type(2)));

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
// two floats to packed bf16, round to nearest even (hardware conversion)
__device__ __forceinline__ uint32_t pack2_rne(float a, float b) {
  const bf16x2_t v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
constexpr bf16x2_t kOnes2 = {(__bf16)1.0f, (__bf16)1.0f};

// v_permlane32_swap(a, b) returns r0 = [a of lanes 0-31 | b of lanes 0-31]
// and r1 = [a of lanes 32-63 | b of lanes 32-63] (lanes 0-31 | 32-63).
// For a value held per lane, r0/r1 of swap(x, x) are the values of the two
// lanes of the pair (l, l^32), in every lane.
// Maxima use the NaN-propagating maximum (v_maximum3_f32): fmaxf would make
// the compiler canonicalise each MFMA result first (one more instruction per
// score pair); no score is NaN.
__device__ __forceinline__ float fmax_nc(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_nc(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t uni_rsrc_a(const void* p, uint32_t n) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return make_rsrc(reinterpret_cast<const void*>(((uint64_t)hi << 32) | lo), __builtin_amdgcn_readfirstlane(n));
}

// Phase boundary: this wavefront's LDS writes are done, then s_barrier; no
// memory access or arithmetic is moved across it.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
constexpr int vmcnt_enc(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// Bytes from the first to the last element of `rows` rows of 128 at stride ld.
__device__ __forceinline__ uint32_t rows_extent(int rows, int64_t ld) {
  return rows > 0 ? (uint32_t)(((rows - 1) * ld + kHd) * 2) : 0u;
}

// ------------------------------------------------- tiles read in both ways
// A tile of 64 rows (keys or queries) of 128 bf16, 256 bytes a row, whose
// 16-byte chunk c of row r is stored at chunk c ^ tile_key(r). Two kinds of
// fragment come out of it without bank conflicts:
//   * rows as the matrix product's outer index (ds_read_b128: 16 lanes read
//     one chunk of 16 consecutive rows; tile_key is a bijection of r & 15);
//   * rows as the contracted index (ds_read_b64_tr_b16: 32 lanes read 64
//     bytes of four consecutive rows, whose keys differ in the bits that
//     pick one of the four 64-byte quarters).
__device__ __forceinline__ int tile_key(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

// Offset of this lane's part of the fragment with rows as outer index: row
// lane & 31 of the tile, elements 16 s + 8 (lane >> 5) .. +7. Step s is this
// offset ^ 32 s; 32 rows further are 8192 bytes.
__device__ __forceinline__ uint32_t row_frag_off(int lane) {
  const int r = lane & 31;
  return (uint32_t)(r * 256 + (((lane >> 5) ^ tile_key(r)) << 4));
}

// The fragment with rows as the contracted index, 32 columns from 32 db and
// 16 rows from 16 s2: ds_read_b64_tr_b16 gives lane i of 16 the elements
// (rows j = 0..3, column i) of the 4 x 16 block whose row j lies at the
// addresses of lanes 4 j .. 4 j + 3, 8 bytes each. Slot 4 h + j of lane half
// lh is row 16 s2 + 8 h + 4 lh + j: the rows that an accumulator of the
// product before holds in its elements 8 s2 + 4 h + j, so that those, packed,
// are the other operand as they stand. Offset for db = 0, s2 = 0, h = 0; db is
// this offset ^ 64 db, h = 1 the offset ^ 32 (tile_key of r + 8) + 2048, s2
// adds 4096.
__device__ __forceinline__ uint32_t col_frag_off(int lane) {
  const int s = lane & 15, r = 4 * (lane >> 5) + (s >> 2);
  const int chunk = 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
  return (uint32_t)(r * 256 + ((chunk ^ tile_key(r)) << 4) + ((s & 1) << 3));
}

// LDS addresses. A tile starts at a multiple of 256 bytes, so the XORs above
// may be applied to the whole address.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) f32x2 lds_f32x2;
typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_addr(const char* p) { return (uint32_t)(uintptr_t)(const lds_char*)p; }
__device__ __forceinline__ bf16x8 row_frag(uint32_t addr, int s) {
  return *reinterpret_cast<const lds_bf16x8*>((uintptr_t)(addr ^ (uint32_t)(32 * s)));
}
__device__ __forceinline__ bf16x8 col_frag(uint32_t addr, int db, int s2) {
  struct Pair { s16x4 a, b; } p;
  const uint32_t x = addr ^ (uint32_t)(64 * db);
  p.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(x + 4096 * s2));
  p.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((x ^ 32) + 4096 * s2 + 2048));
  return __builtin_bit_cast(bf16x8, p);
}

}  // namespace glt

// Device helpers shared by the attention kernels (attention.hip,
// attention_train.hip, attention_bwd.hip).
#pragma once

#include "common.hpp"

namespace glt {

constexpr int kHd = 128;          // head dimension

// Refuses what no attention training entry point serves (attention_train.hip).
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
// A tile of 64 rows (keys or queries) of 128 bf16 in LDS, in groups of four rows
// of 1 KB and 16 bytes between them. In a group the 64-byte quarters of the
// rows lie row by row, quarter by quarter: 16-byte chunk c of row r is at
//   1040 (r >> 2) + 256 (c >> 2) + 64 (r & 3) + 16 (c & 3).
// Two kinds of fragment come out of it without bank conflicts:
//   * rows as the matrix product's outer index (ds_read_b128: 16 lanes read
//     one chunk of 16 consecutive rows, four groups shifted by 16 bytes each);
//   * rows as the contracted index (ds_read_b64_tr_b16: 32 lanes read one
//     quarter of four consecutive rows, 256 consecutive bytes),
// every step of either at a constant distance from the first, which the read
// instruction holds. (With chunks permuted by XOR, equally free of conflicts,
// the addresses cost 60 of a step's 200 vector instruction slots.) Loads of four
// lanes read 64 consecutive bytes of a row.
constexpr int kGroupB = 1040;                 // four rows
constexpr int kTile = 64;
constexpr int kTileB = 16 * kGroupB;          // 16,640 bytes
// The lane's row in its group and chunk, where lane L of a direct-to-LDS load of
// 1 KB fills bytes 16 L of the group.
__device__ __forceinline__ int group_row(int lane) { return (lane >> 2) & 3; }
__device__ __forceinline__ int group_chunk(int lane) { return 4 * (lane >> 4) + (lane & 3); }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) f32x2 lds_f32x2;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) char lds_char;

// Fragment with rows as outer index: row lane & 31, elements 16 s + 8 (lane >>
// 5) .. +7, from the tile's address + row_frag_off(lane). 32 rows further are
// 8 kGroupB bytes.
__device__ __forceinline__ uint32_t row_frag_off(int lane) {
  const int r = lane & 31;
  return (uint32_t)((r >> 2) * kGroupB + (r & 3) * 64 + (lane >> 5) * 16);
}
__device__ __forceinline__ bf16x8 row_frag(const lds_char* p, int s) {
  return *(const lds_bf16x8*)(p + (s >> 1) * 256 + (s & 1) * 32);
}

// Fragment with rows as the contracted index, 32 columns from 32 db and 16 rows
// from 16 s2: ds_read_b64_tr_b16 gives lane i of 16 the elements (rows j = 0..3,
// column i) of the 4 x 16 block whose row j lies at the addresses of lanes
// 4 j .. 4 j + 3, 8 bytes each. Slot 4 h + j of lane half lh is row
// 16 s2 + 8 h + 4 lh + j: the rows that an accumulator of the product before
// holds in its elements 8 s2 + 4 h + j, so that those, packed, are the other
// operand as they stand. From the tile's address + col_frag_off(lane).
__device__ __forceinline__ uint32_t col_frag_off(int lane) {
  const int s = lane & 15;
  return (uint32_t)((lane >> 5) * kGroupB + (s >> 2) * 64 + ((lane >> 4) & 1) * 32 + (s & 3) * 8);
}
__device__ __forceinline__ bf16x8 col_frag(const lds_char* p, int db, int s2) {
  struct Pair { s16x4 a, b; } f;
  lds_char* x = const_cast<lds_char*>(p) + 256 * db + 4 * s2 * kGroupB;
  f.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)x);
  f.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + 2 * kGroupB));
  return __builtin_bit_cast(bf16x8, f);
}

// ------------------------------------------------------ training kernels
// (attention_train.hip, attention_bwd.hip) A wavefront owns 32 rows, in
// registers, and walks tiles of the others.
constexpr float kLog2e = 1.4426950408889634f;

// Sequence b's length in a batch padded to T.
__device__ __forceinline__ int seq_len(const int32_t* seq_lens, int b, int T) {
  return seq_lens ? min(max(seq_lens[b], 0), T) : T;
}

// One tile (64 rows of a head, from byte row0_bytes) into LDS, by this
// wavefront's share of the 16 loads of 1 KB (a group of four rows each). off:
// this lane's byte offset of its first load (tile_lane_off). Rows past the
// descriptor are zeros.
template <int WAVES>
__device__ __forceinline__ void load_tile(__amdgpu_buffer_rsrc_t r, lds_char* dst, int wave, uint32_t off, uint32_t row_bytes,
                                          uint32_t row0_bytes) {
#pragma unroll
  for (int i = 0; i < 16 / WAVES; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + (WAVES * i + wave) * kGroupB), 16,
                                             off + (row0_bytes + 4 * WAVES * i * row_bytes), 0, 0, 0);
}
__device__ __forceinline__ uint32_t tile_lane_off(int wave, int lane, uint32_t row_bytes) {
  return (uint32_t)(4 * wave + group_row(lane)) * row_bytes + (uint32_t)(group_chunk(lane) * 16);
}

// A wavefront's 32 rows of 128 as MFMA operands: lane row (lane & 31),
// elements 16 s + 8 (lane >> 5) .. +7; rows at or past the end are zeros.
__device__ __forceinline__ void load_rows(bf16x8* f, const uint16_t* row, bool live, int lh) {
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const u32x4 x = live ? *reinterpret_cast<const u32x4*>(row + 16 * s + 8 * lh) : u32x4{0u, 0u, 0u, 0u};
    f[s] = __builtin_bit_cast(bf16x8, x);
  }
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// elements 8 s2 .. +7 of an accumulator, rounded: the operand of 16 contracted
// rows in the order that col_frag() reads them
__device__ __forceinline__ bf16x8 pack_frag(const f32x16& x, int s2) {
  const int o = 8 * s2;
  return __builtin_bit_cast(bf16x8, u32x4{pack2_rne(x[o], x[o + 1]), pack2_rne(x[o + 2], x[o + 3]),
                                          pack2_rne(x[o + 4], x[o + 5]), pack2_rne(x[o + 6], x[o + 7])});
}

// Score product of 32 walked rows: x += X . f^T over the 128 columns, the
// fragments read AHEAD steps ahead; between(i) is arithmetic that the
// scheduler may put beside step i's matrix instruction. (The fence per step
// keeps the reads from all being hoisted, which needs more registers than
// there are.)
template <int AHEAD, typename F>
__device__ __forceinline__ void score_product(const lds_char* X, const bf16x8* f, f32x16& x, F between) {
  bf16x8 xa[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) xa[i] = row_frag(X, i);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x = mfma(xa[i % AHEAD], f[i], x);
    if (i + AHEAD < 8) xa[i % AHEAD] = row_frag(X, i + AHEAD);
    between(i);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// an address that is worked out where it is used, not kept in a register for
// every offset
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Accumulator of a transposed product (lane: owned row, elements: d = 32 db +
// 8 g + 4 lh + e) times `scale`, rounded once, to this lane's output row.
__device__ __forceinline__ void store_rows(uint16_t* row, const f32x16* acc, float scale, int lh) {
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const u32x2a w = {pack2_rne(acc[db][4 * g] * scale, acc[db][4 * g + 1] * scale),
                        pack2_rne(acc[db][4 * g + 2] * scale, acc[db][4 * g + 3] * scale)};
      *reinterpret_cast<u32x2a*>(row + 32 * db + 8 * g + 4 * lh) = w;
    }
}

}  // namespace glt

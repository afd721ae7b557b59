// Layout of the 8-bit cache of keys and values (kv8.hip, kv8_attention.hip).
#pragma once

#include "common.hpp"
#include "overlap.hpp"

namespace glt {

// The cache of one layer is a pool of pages of 64 tokens; a page holds its kv
// heads one after the other, each in kHeadB bytes:
//   0       codes of k, [64 tokens][128]
//   8192    codes of v, [128 channels][64 tokens], token t at byte v_byte(t)
//   16384   steps of k, bf16 [64 tokens]
//   16512   steps of v, bf16 [64 tokens]
// A value is code * step, a step for each token, head and tensor. Both products of
// attention read 16 codes of one row that are next to each other in memory: k's
// rows are tokens (scores contract channels), v's are channels (the output
// contracts tokens).
constexpr int kPage = 64;
constexpr int kKv8Hd = 128;
constexpr int kVOff = 8192, kKStepOff = 16384, kVStepOff = 16512;
constexpr int kHeadB = 16640;

// Bits 2 and 3 of the token change places: 8 bytes then hold the eight tokens
// that one lane's accumulators of a 32-row score product hold (tokens 16 s + 8 i
// + 4 lh + e for i = 0, 1 and e = 0..3).
__host__ __device__ constexpr int v_byte(int t) { return (t & 0x33) | ((t & 4) << 1) | ((t & 8) >> 1); }

// Refuses caches and page tables that no entry point serves (kv8.hip).
glt_status check_kv8(const glt_kv8_cache* c, const glt_kv8_seqs* s, const char* who);
// Refuses results (n of them) in the page table and lengths, which workgroups read after
// others have written: a length that changed would lead past what was sized by it.
glt_status check_spared(const glt_kv8_seqs* s, const ByteRows* to, int n, const char* who);
inline ByteRows table_bytes(const int32_t* pages, int64_t rows, int64_t ld, int64_t n) { return {pages, rows, 4 * n, 4 * ld}; }

// Tokens that sequence b holds and how many of them are the call's new ones.
struct Kv8Len { int len, fresh; };
__device__ __forceinline__ Kv8Len kv8_len(const glt_kv8_seqs& s, int b) {
  const int len = min(max(s.lens[b], 0), s.n_table * kPage);
  return {len, min(s.new_lens ? max(s.new_lens[b], 0) : s.T, min(s.T, len))};
}

}  // namespace glt

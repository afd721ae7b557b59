// Keys and values into a paged 8-bit cache and back, for gfx950.
//
//   step = bf16(max |x| / 127) of a token's head, in [2^-100, 2^121]
//   code = x / step, rounded to the nearest whole number
//
// One workgroup per (page that the call touches, kv head, sequence): 16 lanes
// read a row of 256 bytes, a thread the same 8 channels of four consecutive
// tokens, so that it holds the four bytes that lie together in v's transposed
// codes. Those cross LDS into 16-byte stores (whole groups of tokens) or go out
// byte by byte (a page's other tokens are never read or written: other streams
// may hold them).
//
// Bound by memory: 8 sequences of up to 4096 new tokens, 8 kv heads: written in 26 us,
// read back in 23 (269 MB in all, 5.5 TB/s); one token of 64 sequences 6 and 3.5, the
// chain of lengths, table and rows.
#include "kv8.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

struct Kv8Args {
  uint8_t* cache;
  int64_t n_pages;
  glt_kv8_seqs s;
  uint16_t* k;      // read's results, write's inputs
  uint16_t* v;
  int64_t k_ld, v_ld;
  int Hkv;
};

// Byte of a 16-byte chunk m (tokens 16 m .. + 15) of channel d of the
// transposed codes in LDS: chunks permuted so that the 16 lanes of a row, 8
// channels apart, spread over the banks.
__device__ __forceinline__ int lds_chunk(int d, int m) { return d * kPage + ((m ^ ((d >> 3) & 3)) << 4); }

// The sequence's block: page and tokens of the block that are new.
struct Block { uint8_t* at; int first, lo, hi; };  // token of new index 0 in the page; new tokens of the page
__device__ __forceinline__ bool find_block(const Kv8Args& a, int b, Kv8Len n, int i, int64_t* page, int* first) {
  const int start = n.len - n.fresh, pi = start / kPage + i;
  *first = start - pi * kPage;
  *page = pi < a.s.n_table ? a.s.pages[b * a.s.pages_ld + pi] : -1;
  return *page >= 0 && *page < a.n_pages;
}

// Codes of 8 bf16 and the row's step, over the row's 16 lanes.
__device__ __forceinline__ u32x2 row_codes(u32x4 x, uint32_t* step_bits) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  // No bf16 over 127 comes near the middle of two bf16 (127 is odd), so the
  // product with 1 / 127 rounds as the quotient does.
  const float step = fminf(fmaxf(bf16_to_f32(f32_to_bf16(bf16_to_f32((uint16_t)top) * (1.0f / 127.0f))), 0x1p-100f), 0x1p121f);
  const bool bad = top >= 0x7f80u;  // infinity or NaN in the row
  *step_bits = bad ? 0x7fc0u : __float_as_uint(step) >> 16;
  const float inv = __builtin_amdgcn_rcpf(step);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = __uint_as_float(i & 1 ? x[i >> 1] & 0xffff0000u : x[i >> 1] << 16);
    // x / step may lie halfway between two codes, where the product with the
    // reciprocal does not: one step of the remainder makes the quotient exact
    float y = f * inv;
    y = __builtin_fmaf(__builtin_fmaf(-y, step, f), inv, y);
    const int c = (int)__builtin_rintf(fminf(fmaxf(y, -127.f), 127.f));
    w[i >> 2] |= (uint32_t)(c & 0xff) << (8 * (i & 3));
  }
  return bad ? u32x2{0u, 0u} : u32x2{w[0], w[1]};
}

// byte e of four words
__device__ __forceinline__ uint32_t gather_byte(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int e) {
  return ((a >> (8 * e)) & 0xff) | (((b >> (8 * e)) & 0xff) << 8) | (((c >> (8 * e)) & 0xff) << 16) |
         (((d >> (8 * e)) & 0xff) << 24);
}

__global__ void __launch_bounds__(256) kv8_write_kernel(const Kv8Args a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kKv8Hd * kPage];
  const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Kv8Len n = kv8_len(a.s, b);
  int64_t page;
  int first;
  if (!find_block(a, b, n, blockIdx.x, &page, &first)) return;
  const int lo = max(first, 0), hi = min(first + n.fresh, kPage);  // the page's tokens that this call writes
  if (lo >= hi) return;
  uint8_t* at = a.cache + (page * a.Hkv + h) * kHeadB;
  const int row = 4 * (tid >> 4), c = tid & 15;  // tokens row .. + 3 of the page, channels 8 c .. + 7
  u32x4 kx[4], vx[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = row + j >= lo && row + j < hi;
    const int64_t tok = (int64_t)b * a.s.T + (row + j - first);
    kx[j] = in ? *reinterpret_cast<const u32x4*>(a.k + tok * a.k_ld + h * kKv8Hd + 8 * c) : u32x4{0u, 0u, 0u, 0u};
    vx[j] = in ? *reinterpret_cast<const u32x4*>(a.v + tok * a.v_ld + h * kKv8Hd + 8 * c) : u32x4{0u, 0u, 0u, 0u};
  }
  uint32_t step[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u32x2 w = row_codes(kx[j], &step[j]);
    if (row + j >= lo && row + j < hi) {
      *reinterpret_cast<u32x2*>(at + (row + j) * kKv8Hd + 8 * c) = w;
      if (c == 0) *reinterpret_cast<uint16_t*>(at + kKStepOff + 2 * (row + j)) = (uint16_t)step[j];
    }
  }
  u32x2 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = row_codes(vx[j], &step[j]);
    if (row + j >= lo && row + j < hi && c == 0) *reinterpret_cast<uint16_t*>(at + kVStepOff + 2 * (row + j)) = (uint16_t)step[j];
  }
  const int q = v_byte(row);  // the four tokens' bytes are q .. q + 3
  if (hi - lo < 4) {  // a step or two of generation
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (row + j >= lo && row + j < hi)
#pragma unroll
        for (int e = 0; e < 8; ++e) at[kVOff + (8 * c + e) * kPage + q + j] = (uint8_t)(w[j][e >> 2] >> (8 * (e & 3)));
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    *reinterpret_cast<uint32_t*>(lds + lds_chunk(8 * c + e, q >> 4) + (q & 15)) =
        gather_byte(w[0][e >> 2], w[1][e >> 2], w[2][e >> 2], w[3][e >> 2], e & 3);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = (tid + 256 * i) >> 2, m = tid & 3;
    const u32x4 x = *reinterpret_cast<const u32x4*>(lds + lds_chunk(d, m));
    uint8_t* to = at + kVOff + d * kPage + 16 * m;
    if (lo <= 16 * m && hi >= 16 * m + 16) {
      *reinterpret_cast<u32x4*>(to) = x;
      continue;
    }
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      const int t = 16 * m + v_byte(y);  // v_byte is its own inverse
      if (t >= lo && t < hi) to[y] = (uint8_t)(x[y >> 2] >> (8 * (y & 3)));
    }
  }
}

// A code's value, rounded once.
__device__ __forceinline__ uint16_t code_value(uint32_t w, int e, float step) {
  return (uint16_t)(__builtin_bit_cast(uint16_t, (__bf16)((float)(int8_t)(w >> (8 * e)) * step)));
}
__device__ __forceinline__ u32x4 code_values(u32x2 w, float step) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = (uint32_t)code_value(w[i >> 1], 2 * (i & 1), step) | ((uint32_t)code_value(w[i >> 1], 2 * (i & 1) + 1, step) << 16);
  return r;
}

__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Args a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kKv8Hd * kPage];
  const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Kv8Len n = kv8_len(a.s, b);
  int64_t page;
  int first;
  const bool ok = find_block(a, b, n, blockIdx.x, &page, &first);
  const int lo = max(first, 0), hi = min(first + n.fresh, kPage);  // the page's tokens to read
  const int end = min(first + a.s.T, kPage);                       // rows behind them get zeros
  if (lo >= end) return;
  const uint8_t* at = a.cache + ((ok ? page : 0) * a.Hkv + h) * kHeadB;
  const int row = 4 * (tid >> 4), c = tid & 15;
  u32x2 kw[4];
  float ks[4], vs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kw[j] = u32x2{0u, 0u};
    ks[j] = vs[j] = 0.f;
    if (row + j >= lo && row + j < hi) {
      kw[j] = *reinterpret_cast<const u32x2*>(at + (row + j) * kKv8Hd + 8 * c);
      ks[j] = ok ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(at + kKStepOff + 2 * (row + j))) : NAN;
      vs[j] = ok ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(at + kVStepOff + 2 * (row + j))) : NAN;
    }
  }
  if (lo < hi) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = (tid + 256 * i) >> 2, m = tid & 3;
      if (lo < 16 * m + 16 && hi > 16 * m)
        *reinterpret_cast<u32x4*>(lds + lds_chunk(d, m)) = *reinterpret_cast<const u32x4*>(at + kVOff + d * kPage + 16 * m);
    }
  }
  __syncthreads();
  const int q = v_byte(row);
  uint32_t t[8];  // a channel's four tokens
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = *reinterpret_cast<const uint32_t*>(lds + lds_chunk(8 * c + e, q >> 4) + (q & 15));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (row + j < lo || row + j >= end) continue;
    const int64_t tok = (int64_t)b * a.s.T + (row + j - first);
    *reinterpret_cast<u32x4*>(a.k + tok * a.k_ld + h * kKv8Hd + 8 * c) = code_values(kw[j], ks[j]);
    const bool live = row + j < hi;  // what LDS holds elsewhere is not looked at
    const u32x2 vw = {live ? gather_byte(t[0], t[1], t[2], t[3], j) : 0u, live ? gather_byte(t[4], t[5], t[6], t[7], j) : 0u};
    *reinterpret_cast<u32x4*>(a.v + tok * a.v_ld + h * kKv8Hd + 8 * c) = code_values(vw, vs[j]);
  }
}

// Caches that page ids and offsets reach.
bool cache_sizes(int64_t n_pages, int n_kv_heads) {
  return n_pages > 0 && n_pages <= INT32_MAX && n_kv_heads > 0 && n_kv_heads <= 4096;
}

// pages that T tokens from any place of a page lie in
int64_t token_pages(const glt_kv8_seqs* s) { return (s->T + 2 * kPage - 2) / kPage; }

glt_status check_tokens(const glt_kv8_cache* c, const glt_kv8_seqs* s, const void* k, int64_t k_ld, const void* v,
                        int64_t v_ld, const char* who) {
  const int64_t lds[2] = {k_ld, v_ld};
  for (int i = 0; i < 2; ++i)
    GLT_CHECK(lds[i] >= (int64_t)c->n_kv_heads * kKv8Hd && lds[i] % 8 == 0 && lds[i] < ((int64_t)1 << 31), GLT_ERR_SHAPE,
              "%s: %c_ld %lld (at least %d heads of %d, a multiple of 8)", who, "kv"[i], (long long)lds[i], c->n_kv_heads, kKv8Hd);
  GLT_CHECK(k && v, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(((uintptr_t)k | (uintptr_t)v) % 16 == 0, GLT_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", who);
  // a launch holds less than 2^32 threads, 256 for a page and head
  GLT_CHECK(token_pages(s) * s->B < (1 << 24) / c->n_kv_heads, GLT_ERR_SHAPE, "%s: B=%d T=%d n_kv_heads=%d", who, s->B, s->T,
            c->n_kv_heads);
  return GLT_OK;
}

Kv8Args pack_args(const glt_kv8_cache* c, const glt_kv8_seqs* s, void* k, int64_t k_ld, void* v, int64_t v_ld) {
  Kv8Args a{};
  a.cache = static_cast<uint8_t*>(c->data);
  a.n_pages = c->n_pages;
  a.s = *s;
  a.k = static_cast<uint16_t*>(k);
  a.v = static_cast<uint16_t*>(v);
  a.k_ld = k_ld;
  a.v_ld = v_ld;
  a.Hkv = c->n_kv_heads;
  return a;
}
dim3 token_grid(const glt_kv8_cache* c, const glt_kv8_seqs* s) {
  return dim3((unsigned)token_pages(s), (unsigned)c->n_kv_heads, (unsigned)s->B);
}

}  // namespace

glt_status check_kv8(const glt_kv8_cache* c, const glt_kv8_seqs* s, const char* who) {
  GLT_CHECK(c && s, GLT_ERR_INVALID_ARG, "%s: null descriptor", who);
  GLT_CHECK(c->head_dim == kKv8Hd, GLT_ERR_UNSUPPORTED, "%s: head_dim %d (only %d)", who, c->head_dim, kKv8Hd);
  GLT_CHECK(cache_sizes(c->n_pages, c->n_kv_heads), GLT_ERR_SHAPE, "%s: n_pages=%lld n_kv_heads=%d", who,
            (long long)c->n_pages, c->n_kv_heads);
  GLT_CHECK(s->B >= 0 && s->B <= 8192 && s->T >= 0 && s->T <= (1 << 24), GLT_ERR_SHAPE, "%s: B=%d (at most 8192) T=%d", who,
            s->B, s->T);
  GLT_CHECK(s->n_table >= 0 && s->n_table <= (1 << 23) && s->pages_ld >= s->n_table, GLT_ERR_SHAPE,
            "%s: %d pages a sequence, rows %lld apart", who, s->n_table, (long long)s->pages_ld);
  if (s->B == 0 || s->T == 0) return GLT_OK;
  GLT_CHECK(c->data && s->lens && (s->pages || s->n_table == 0), GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK((uintptr_t)c->data % 16 == 0 && ((uintptr_t)s->pages | (uintptr_t)s->lens | (uintptr_t)s->new_lens) % 4 == 0,
            GLT_ERR_ALIGNMENT, "%s: the cache must be 16-byte aligned, tables and lengths 4-byte", who);
  return GLT_OK;
}

glt_status check_spared(const glt_kv8_seqs* s, const ByteRows* to, int n, const char* who) {
  const ByteRows read[] = {table_bytes(s->pages, s->B, s->pages_ld, s->n_table), dense_bytes(s->lens, 4 * (int64_t)s->B),
                           dense_bytes(s->new_lens, s->new_lens ? 4 * (int64_t)s->B : 0)};
  for (int i = 0; i < n; ++i)
    for (const ByteRows& x : read)
      GLT_CHECK(!overlap(to[i], x), GLT_ERR_INVALID_ARG, "%s: results must overlap neither pages nor lengths", who);
  return GLT_OK;
}

}  // namespace glt

using namespace glt;

extern "C" size_t glt_kv8_size(int64_t n_pages, int32_t n_kv_heads, int32_t head_dim) {
  if (!cache_sizes(n_pages, n_kv_heads) || head_dim != kKv8Hd) return 0;
  return (size_t)n_pages * n_kv_heads * kHeadB;
}

extern "C" glt_status glt_kv8_write(const glt_kv8_cache* c, const glt_kv8_seqs* s, const void* k, int64_t k_ld, const void* v,
                                    int64_t v_ld, void* stream) {
  glt_status r = check_kv8(c, s, "glt_kv8_write");
  if (r != GLT_OK || s->B == 0 || s->T == 0) return r;
  r = check_tokens(c, s, k, k_ld, v, v_ld, "glt_kv8_write");
  if (r != GLT_OK) return r;
  const int64_t tokens = (int64_t)s->B * s->T, w = 2 * kKv8Hd * (int64_t)c->n_kv_heads;
  const ByteRows pool = dense_bytes(c->data, (int64_t)glt_kv8_size(c->n_pages, c->n_kv_heads, c->head_dim));
  GLT_CHECK(!overlap(pool, {k, tokens, w, 2 * k_ld}) && !overlap(pool, {v, tokens, w, 2 * v_ld}), GLT_ERR_INVALID_ARG,
            "glt_kv8_write: k and v must not overlap the cache");
  r = check_spared(s, &pool, 1, "glt_kv8_write");
  if (r != GLT_OK) return r;
  const Kv8Args a = pack_args(c, s, const_cast<void*>(k), k_ld, const_cast<void*>(v), v_ld);
  GLT_LAUNCH("kv8_write", kv8_write_kernel, token_grid(c, s), dim3(256), 0, as_stream(stream), a);
  GLT_LAUNCH_CHECK("kv8_write");
  return GLT_OK;
}

extern "C" glt_status glt_kv8_read(const glt_kv8_cache* c, const glt_kv8_seqs* s, void* k, int64_t k_ld, void* v, int64_t v_ld,
                                   void* stream) {
  glt_status r = check_kv8(c, s, "glt_kv8_read");
  if (r != GLT_OK || s->B == 0 || s->T == 0) return r;
  r = check_tokens(c, s, k, k_ld, v, v_ld, "glt_kv8_read");
  if (r != GLT_OK) return r;
  const int64_t tokens = (int64_t)s->B * s->T, w = 2 * kKv8Hd * (int64_t)c->n_kv_heads;
  const ByteRows pool = dense_bytes(c->data, (int64_t)glt_kv8_size(c->n_pages, c->n_kv_heads, c->head_dim));
  const ByteRows to[] = {{k, tokens, w, 2 * k_ld}, {v, tokens, w, 2 * v_ld}};
  GLT_CHECK(!overlap(pool, to[0]) && !overlap(pool, to[1]) && !overlap(to[0], to[1]), GLT_ERR_INVALID_ARG,
            "glt_kv8_read: k and v must overlap neither the cache nor each other");
  r = check_spared(s, to, 2, "glt_kv8_read");
  if (r != GLT_OK) return r;
  const Kv8Args a = pack_args(c, s, k, k_ld, v, v_ld);
  GLT_LAUNCH("kv8_read", kv8_read_kernel, token_grid(c, s), dim3(256), 0, as_stream(stream), a);
  GLT_LAUNCH_CHECK("kv8_read");
  return GLT_OK;
}

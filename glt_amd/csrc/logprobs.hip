// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and the gradient of the first two.
//
//   z = x / temperature, lse = log sum exp z, logp_v = z_v - lse, p = exp logp
//   entropy H = -sum p logp = lse - sum p z
//   d logp_id / dz_v = [v = id] - p_v,  dH / dz_v = -p_v (logp_v + H)
//
// Everything is read once and bound by HBM: 2 or 4 bytes a logit forward, twice
// that backward, against about ten vector instructions (a copy of 1 GiB reaches
// 5.1 TB/s).
//
// Forward: one workgroup of four wavefronts per piece of a row (32 KB, held in
// registers: eight 16-byte chunks a thread, chunk k of thread t being chunk
// 256 k + t), each wavefront leaving its maximum, sum exp and sum z exp, and the
// workgroup its k largest logits; a workgroup per row then joins the row's
// parts in their order, in 64 bits, and merges the lists. The cut depends on V
// alone, so a row has the same bits in every call, and a single row still spreads
// over V / 16384 workgroups (bf16; half as many logits a piece in f32).
// 4096 x 128256 bf16: 176 to 190 us without alternatives (5.5 to 6.0 TB/s), 200
// with 5, 216 with 20, 260 with 64; 2048 x 128256 f32: 178 us (5.9 TB/s), 189 with
// 20. Seven rows of f32 with 20: 8 + 6 us, the latency of its steps.
// Not fast: alternatives of rows in which nearly all logits are equal, masked ones
// too. Their pieces are left to the row's one workgroup (piece_top_any): with
// 100 allowed tokens and 20 alternatives 4096 rows of bf16 take 2780 us, seven of
// f32 1190 (183 and 17 without alternatives).
//
// In log2 units c = log2(e) / temperature: a wavefront's terms are exp2((x - m)
// c) of its maximum m, and the joined sum is told m c in 64 bits, where the
// product is exact. Where |m c| is below kShiftMax they are formed as
// exp2(fma(x, c, -shift)) with the rounded shift m c, an instruction less (4096
// x 128256 bf16 with 20 alternatives: 216 us, otherwise 229), and put right
// afterwards: left as they are, a certain token's log probability comes out
// above 0, and past |m c| = 2^31 the rounding is beyond exp2's range.
#include <atomic>
#include <cmath>

#include "common.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kChunks = 8;                       // 16-byte chunks a thread holds
constexpr int kMaxTop = 64;                      // alternatives at most: one per lane of the selecting wavefront
constexpr int kMaxIds = 64;
constexpr int kMaxV = 1 << 20;
constexpr int kCap = 1024;                       // candidates of a piece held in LDS
constexpr int kLdsFree = 60 * 1024;              // dynamic LDS that needs no leave, beside RowList
constexpr int kHitCap = 128;                     // chunks of a piece that hold candidates
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453094;
constexpr float kShiftMax = 0x1p20f;             // rounded to 2^-5 at least

// 16 bytes of logits at any element address (gfx950 loads and stores
// unaligned vectors; rows of an odd vocabulary start anywhere)
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T>
struct Elems;
template <>
struct Elems<uint16_t> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float get(const u32x4& c, int e) {
    return (e & 1) ? __uint_as_float(c[e >> 1] & 0xFFFF0000u) : __uint_as_float(c[e >> 1] << 16);
  }
  static constexpr uint32_t neg_inf = 0xFF80u;
  static __device__ __forceinline__ void put(u32x4& c, int e, uint32_t bits) { c[e >> 1] |= bits << (16 * (e & 1)); }
};
template <>
struct Elems<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ float get(const u32x4& c, int e) { return __uint_as_float(c[e]); }
  static constexpr uint32_t neg_inf = 0xFF800000u;
  static __device__ __forceinline__ void put(u32x4& c, int e, uint32_t bits) { c[e] = bits; }
};
// The maxima of a thread's chunks; two a register where they are bf16 values.
template <typename T>
struct Maxima {
  static constexpr int per = 4 / sizeof(T);
  uint32_t w[kChunks / per];
  __device__ __forceinline__ void set(int q, float v) {
    const uint32_t u = __float_as_uint(v);
    if constexpr (per == 1) w[q] = u;
    else w[q / 2] = q & 1 ? w[q / 2] | (u & 0xFFFF0000u) : u >> 16;
  }
  __device__ __forceinline__ float get(int q) const {
    if constexpr (per == 1) return __uint_as_float(w[q]);
    else return __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
  }
};
template <typename T>
constexpr int kPiece = kThreads * kChunks * Elems<T>::n;  // logits per workgroup

__device__ __forceinline__ uint32_t bits_of(uint16_t v) { return v; }
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ float value_of(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float value_of(float v) { return v; }

// Chunk of a row from element e; elements at or past V are -inf.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int e, int V) {
  using E = Elems<T>;
  if (e + E::n <= V) return *reinterpret_cast<const u32x4_any*>(row + e);
  constexpr uint32_t inf = sizeof(T) == 2 ? E::neg_inf * 0x10001u : E::neg_inf;
  if (e >= V) return u32x4{inf, inf, inf, inf};
  u32x4 c = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < E::n; ++j) {
    const uint32_t b = bits_of(row[min(e + j, V - 1)]);  // in place of what lies past the row
    E::put(c, j, e + j < V ? b : E::neg_inf);
  }
  return c;
}

// Order-preserving integer of a float's bits (NaN beyond the infinities; both
// zeros are one value).
__device__ __forceinline__ uint32_t ord(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ord(uint32_t o) {
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
// Key of a candidate: larger is better, the lower index among equal values.
__device__ __forceinline__ uint64_t make_key(uint32_t o, uint32_t index) { return (uint64_t)o << 32 | (0xFFFFFFFFu - index); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Which piece of all rows (row by row) a workgroup takes. Workgroups are dealt
// round-robin over the eight XCDs; in plain order two, four or eight pieces a row
// would give each XCD always the same pieces, the short last ones to one or two
// of them, and the rows of one parity, of which an odd vocabulary makes one half
// slower (4096 x 50001 bf16, four pieces: 108 us in plain order, 88 so; 79 for an
// even row stride).
// Here an XCD takes eight consecutive pieces of every 64, the eights handed on
// by one from 64 to 64.
__device__ __forceinline__ uint32_t piece_index(uint32_t block, uint32_t blocks) {
  const uint32_t g = block / 64, x = block % 8, j = block / 8 % 8;
  return g * 64 + 64 > blocks ? block : g * 64 + 8 * ((x + g) % 8) + j;
}

// A wavefront's part of a row: sum of exp2(a - shift) and of (a - shift)
// exp2(a - shift) over its logits, a = x c.
struct Part {
  double shift;
  float s, t;
};

template <int CAP>
struct KeyList {
  static constexpr uint32_t cap = CAP;
  uint32_t count;
  uint32_t sums[kWaves];
  uint64_t cand[CAP];
};
struct TopLds : KeyList<kCap> {
  uint32_t group[kWaves][64];
  uint32_t tau, hits, bad;
  uint32_t hit_at[kHitCap];
};
using RowList = KeyList<kMaxTop>;

// Appends the lanes' keys where `hit`: one LDS atomic per wavefront. (The list's
// order is not fixed; what is made of it goes by the keys, no two of which are
// equal.)
template <typename List>
__device__ __forceinline__ void append(List& L, bool hit, uint64_t key) {
  const uint64_t mask = __ballot(hit);
  if (!mask) return;
  const int lane = threadIdx.x & 63, first = __ffsll((unsigned long long)mask) - 1;
  uint32_t base = 0;
  if (lane == first) base = atomicAdd(&L.count, (uint32_t)__popcll(mask));
  const uint32_t at = __shfl(base, first) + __popcll(mask & ((1ull << lane) - 1));
  if (hit && at < List::cap) L.cand[at] = key;
}

// Sum over the NT threads of a count (all threads get it).
template <int NT>
__device__ __forceinline__ uint32_t block_count(RowList& L, uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) L.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) t += L.sums[w];
  return t;
}

// The k largest of n keys in L.cand, in order, to out[0, k), by counting; a piece
// of fewer than k logits leaves zeros, which are below every key.
template <int NT, typename List>
__device__ __forceinline__ void rank_keys(const List& L, uint32_t n, int k, uint64_t* out) {
  for (uint32_t i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = L.cand[i];
    uint32_t r = 0;
    for (uint32_t j = 0; j < n; ++j) r += L.cand[j] > key;
    if (r < (uint32_t)k) out[r] = key;
  }
  for (uint32_t i = n + threadIdx.x; i < (uint32_t)k; i += NT) out[i] = 0;
}

// First key of a piece whose list piece_top() left to piece_top_any(). (A logit
// that has this key, a NaN, costs its piece that second look.)
constexpr uint64_t kUnranked = ~0ull;

// The k largest logits of a piece, in order, as keys to out[0, k).
// cm: the maxima of the thread's chunks, nan: the thread saw one (or +inf).
//
// A bound first: the k-th largest of the threads' maxima is at most the k-th
// largest logit, and a few more than k logits reach it (256 ln(256 / (256 - k))
// for logits in random order: 21 for k = 20, 74 for 64); one wavefront finds it
// by bisection over the bits. The chunks whose maximum reaches it are listed,
// their logits read again side by side, and those that reach it ranked by
// counting. A piece whose lists overflow, or that holds a NaN, is marked for
// piece_top_any().
template <typename T>
__device__ __forceinline__ void piece_top(const T* x, const Maxima<T>& cm, bool nan, int e0, int V, int k, uint64_t* out, TopLds& L) {
  using E = Elems<T>;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // the chunks' places are worked out again, not kept since their loads
  const int lane = tid & 63, wave = threadIdx.x >> 6;
  float m = cm.get(0);
#pragma unroll
  for (int q = 1; q < kChunks; ++q) m = fmaxf(m, cm.get(q));
  L.group[wave][lane] = ord(m);
  if (tid == 0) L.hits = L.count = L.bad = 0;
  __syncthreads();
  if (nan) L.bad = 1;
  if (wave == 0) {
    uint32_t g[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) g[w] = L.group[w][lane];
    // the largest value that at least k threads' maxima reach
    constexpr int low = sizeof(T) == 2 ? 16 : 0;
    uint32_t tau = 0;
#pragma unroll 1
    for (int b = 31; b >= low; --b) {
      const uint32_t y = tau | (1u << b);
      int reach = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) reach += __popcll(__ballot(g[w] >= y));
      if (reach >= k) tau = y;
    }
    // bf16: the low half of ord() follows from the sign
    if (low && !(tau & 0x80000000u)) tau |= 0xFFFFu;
    if (lane == 0) L.tau = max(tau, 0x007FFFFFu);  // -inf
  }
  __syncthreads();
  const float tf = from_ord(L.tau);
#pragma unroll
  for (int q = 0; q < kChunks; ++q) {
    const int e = e0 + (q * kThreads + tid) * E::n;
    const bool in = cm.get(q) >= tf && e < V;
    const uint64_t mask = __ballot(in);
    if (!mask) continue;
    const int first = __ffsll((unsigned long long)mask) - 1;
    uint32_t base = 0;
    if (lane == first) base = atomicAdd(&L.hits, (uint32_t)__popcll(mask));
    const uint32_t at = __shfl(base, first) + __popcll(mask & ((1ull << lane) - 1));
    if (in && at < kHitCap) L.hit_at[at] = e;
  }
  __syncthreads();
  const uint32_t hits = L.hits;
  if (hits > kHitCap || L.bad) {
    if (tid == 0) out[0] = kUnranked;
    return;
  }
  for (uint32_t i = tid; i < (hits * E::n + 63) / 64 * 64; i += kThreads) {
    bool in = i < hits * E::n;
    const uint32_t e = in ? L.hit_at[i / E::n] + i % E::n : 0u;
    in = in && e < (uint32_t)V;
    const float v = in ? value_of(x[e]) : 0.f;
    append(L, in && v >= tf, make_key(ord(v), e));
  }
  __syncthreads();
  rank_keys<kThreads>(L, L.count, k, out);  // at most kHitCap chunks of 8: no more than kCap
}
static_assert(kHitCap * 8 <= kCap, "the listed chunks' logits fit the candidates' list");

// The same for any piece, however many logits are equal and whatever NaNs it
// holds (they rank by their bits): the k-th largest key by bisection over its
// value's bits; the keys above that value, then the equal ones by index.
template <typename T, int NT>
__device__ void piece_top_any(const T* x, int e0, int V, int k, uint64_t* out, RowList& L) {
  using E = Elems<T>;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int end = min(V, e0 + kPiece<T>);
  const uint32_t want = min(k, end - e0);
  constexpr int low = sizeof(T) == 2 ? 16 : 0, steps = kChunks * kThreads / NT;
  // counts of the logits whose ord() is at least / above a value
  auto count = [&](uint32_t o, bool above) {
    uint32_t v = 0;
#pragma unroll 1
    for (int q = 0; q < steps; ++q) {
      const int e = e0 + (q * NT + tid) * E::n;
      const u32x4 y = load_chunk(x, e, V);
#pragma unroll
      for (int j = 0; j < E::n; ++j) {
        const uint32_t z = ord(E::get(y, j));
        v += e + j < V && (above ? z > o : z >= o);
      }
    }
    return block_count<NT>(L, v);
  };
  uint32_t kth = 0;
#pragma unroll 1
  for (int b = 31; b >= low; --b) {
    const uint32_t y = kth | (1u << b);
    if (count(y, false) >= want) kth = y;
  }
  if (low && !(kth & 0x80000000u)) kth |= 0xFFFFu;
  uint32_t have = count(kth, true);  // fewer than want
  __syncthreads();
  if (tid == 0) L.count = 0;
  __syncthreads();
#pragma unroll 1
  for (int q = 0; q < steps; ++q) {
    const int e = e0 + (q * NT + tid) * E::n;
    const u32x4 y = load_chunk(x, e, V);
#pragma unroll
    for (int j = 0; j < E::n; ++j) {
      const uint32_t z = ord(E::get(y, j));
      append(L, e + j < V && z > kth, make_key(z, e + j));
    }
  }
  __syncthreads();
  // equal ones in index order: chunk by chunk, a thread's behind those of the
  // threads before it
#pragma unroll 1
  for (int q = 0; q < steps && have < want; ++q) {
    const int e = e0 + (q * NT + tid) * E::n;
    const u32x4 y = load_chunk(x, e, V);
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < E::n; ++j) mine += e + j < V && ord(E::get(y, j)) == kth;
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t z = __shfl_up(upto, o);
      if (lane >= o) upto += z;
    }
    __syncthreads();
    if (lane == 63) L.sums[wave] = upto;
    __syncthreads();
    uint32_t at = have + upto - mine;
    for (int w = 0; w < wave; ++w) at += L.sums[w];
#pragma unroll
    for (int j = 0; j < E::n; ++j)
      if (e + j < V && ord(E::get(y, j)) == kth) {
        if (at < want) L.cand[at] = make_key(kth, e + j);
        ++at;
      }
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) have += L.sums[w];
  }
  __syncthreads();
  rank_keys<NT>(L, want, k, out);
}

struct FwdArgs {
  const void* logits;
  int64_t ld;
  int rows, V, np, n_ids, k;
  float c;        // log2(e) / temperature
  const int32_t* ids;
  Part* parts;    // [rows, np, kWaves]
  uint64_t* top;  // [rows, np, k]
  float* logprobs;
  float* entropy;
  float* lse;
  int32_t* top_ids;
  float* top_logprobs;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 8) logprobs_piece_kernel(const FwdArgs a) {
  using E = Elems<T>;
  const int tid = threadIdx.x;
  const uint32_t at = piece_index(blockIdx.x, gridDim.x);
  const int64_t row = at / a.np;
  const int piece = (int)(at % a.np), e0 = piece * kPiece<T>;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  u32x4 ch[kChunks];
#pragma unroll
  for (int q = 0; q < kChunks; ++q) ch[q] = load_chunk(x, e0 + (q * kThreads + tid) * E::n, a.V);
  Maxima<T> cm;
  float mn = INFINITY, m = -INFINITY;
#pragma unroll
  for (int q = 0; q < kChunks; ++q) {
    float c = E::get(ch[q], 0);
    mn = __builtin_elementwise_minimum(mn, c);  // of NaN and anything: NaN
#pragma unroll
    for (int j = 1; j < E::n; ++j) {
      c = fmaxf(c, E::get(ch[q], j));
      mn = __builtin_elementwise_minimum(mn, E::get(ch[q], j));
    }
    m = fmaxf(m, c);
    if constexpr (TOP) cm.set(q, c);
    // the chunk is unpacked again below rather than kept so (64 more registers)
    asm volatile("" : "+v"(ch[q]));
  }
  m = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_max(m))));
  Part p;
  p.s = p.t = 0.f;
  const float shift = m * a.c;
  float off = 0.f;  // the fast loop's exponent of the maximum
  // Shifts whose rounding counts and differences so large that 0 * -inf or an
  // overflow could come up are rare enough for a loop of their own: rows and
  // wavefronts masked with a large number, -inf, NaN, the row's end.
  if (__any(!(mn * a.c > -1e37f)) || !(fabsf(shift) < kShiftMax)) {
    if (m == -INFINITY) {  // nothing is allowed, and nothing is added but a NaN, which the maximum passed over
      p.s = mn == mn ? 0.f : mn;
    } else {
#pragma unroll
      for (int q = 0; q < kChunks; ++q)
#pragma unroll
        for (int j = 0; j < E::n; ++j) {
          const float d = (E::get(ch[q], j) - m) * a.c;
          const float arg = d < -200.f ? -200.f : d;  // exp2 of it is 0; NaN stays
          const float e = __builtin_amdgcn_exp2f(arg);
          p.s += e;
          p.t = fmaf(e, arg, p.t);
        }
    }
  } else {
    off = fmaf(m, a.c, -shift);
    float s0 = 0.f, t0 = 0.f;
#pragma unroll
    for (int q = 0; q < kChunks; ++q) {
#pragma unroll
      for (int j = 0; j < E::n; j += 2) {
        const float a0 = fmaf(E::get(ch[q], j), a.c, -shift), a1 = fmaf(E::get(ch[q], j + 1), a.c, -shift);
        const float e0_ = __builtin_amdgcn_exp2f(a0), e1_ = __builtin_amdgcn_exp2f(a1);
        p.s += e0_;
        s0 += e1_;
        p.t = fmaf(e0_, a0, p.t);
        t0 = fmaf(e1_, a1, t0);
      }
      asm volatile("" : "+v"(ch[q]));
    }
    p.s += s0;
    p.t += t0;
  }
  const bool nan = TOP && !(p.s < INFINITY);
  p.s = wave_sum(p.s);
  p.t = wave_sum(p.t);
  if (off != 0.f) {
    // from the rounded shift to m c; as the maximum's term is 1 and no exponent
    // above 0, the sum is at least 1 and the other at most 0
    const float f = __builtin_amdgcn_exp2f(-off);
    p.t = fminf((p.t - off * p.s) * f, 0.f);
    p.s = fmaxf(p.s * f, 1.f);
  }
  p.shift = (double)m * (double)a.c;
  if ((tid & 63) == 0) a.parts[(row * a.np + piece) * kWaves + (tid >> 6)] = p;
  if constexpr (TOP) {
    __shared__ TopLds L;
    piece_top<T>(x, cm, nan, e0, a.V, a.k, a.top + (row * a.np + piece) * a.k, L);
  }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// One workgroup per row: its parts joined in 64 bits (by every wavefront), the
// given tokens' log probabilities, and the pieces' alternatives merged. The
// r-th keys of the np lists, r = ceil(k / np), are np r >= k keys: the least
// of them bounds the k-th from below. What reaches it (70 of 320 keys at V =
// 128256 f32, k = 20) goes to LDS and is ranked by counting. LDS: np * k
// keys. One wavefront where the pieces' lists hold at most 64 keys, else four.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) logprobs_row_kernel(const FwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint64_t keys[];
  __shared__ RowList L;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const Part* parts = a.parts + row * a.np * kWaves;
  const int n = a.np * kWaves;
  double M = -INFINITY;
  for (int i = lane; i < n; i += 64) M = fmax(M, parts[i].shift);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmax(M, __shfl_xor(M, o));
  double s = 0.0, t = 0.0;
  for (int i = lane; i < n; i += 64) {
    const Part p = parts[i];
    if (p.shift == -INFINITY && p.s == 0.f) continue;  // nothing allowed in it
    const double d = p.shift - M, f = d < -1000.0 ? 0.0 : exp2(d);  // (a NaN part stays one)
    s += p.s * f;
    t += (p.t + p.s * d) * f;
  }
  s = wave_sum64(s);
  t = wave_sum64(t);
  const bool none = M == -INFINITY && s == 0.0;  // no token is allowed
  const double l2s = log2(s), l2 = none ? -INFINITY : M + l2s;
  if (tid == 0) {
    if (a.lse) a.lse[row] = (float)(l2 * kLn2);
    if (a.entropy) a.entropy[row] = none ? 0.f : (float)((l2s - t / s) * kLn2);
  }
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  // z - lse in log2 units, where both carry c's rounding alike; the maximum first,
  // beside which a large row's log2 s would be lost
  auto logp = [&](float v) {
    if (v == -INFINITY) return s == s ? -INFINITY : NAN;
    return (float)((((double)v * (double)a.c - M) - l2s) * kLn2);
  };
  if (tid < a.n_ids) {
    const int id = a.ids[row * a.n_ids + tid];
    a.logprobs[row * a.n_ids + tid] = id < 0 ? 0.f : id >= a.V ? NAN : logp(value_of(x[id]));
  }
  if (a.k == 0) return;
  const int nk = a.np * a.k;
  uint64_t* top = a.top + row * nk;
  for (int p0 = 0; p0 < a.np; p0 += 64) {
    uint64_t left = __ballot(p0 + lane < a.np && top[min(p0 + lane, a.np - 1) * a.k] == kUnranked);
    while (left) {
      const int p = p0 + __ffsll((unsigned long long)left) - 1;
      left &= left - 1;
      __syncthreads();  // every wavefront has seen the marks
      piece_top_any<T, NT>(x, p * kPiece<T>, a.V, a.k, top + p * a.k, L);
      __syncthreads();
    }
  }
  const int r1 = (a.k + a.np - 1) / a.np - 1;
  uint64_t bound = ~0ull;
  for (int i = lane; i < a.np; i += 64) bound = min(bound, top[i * a.k + r1]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t y = (uint64_t)__shfl_xor((unsigned long long)bound, o);
    bound = min(bound, y);
  }
  if (tid == 0) L.count = 0;
  __syncthreads();
  for (int i = tid; i < nk; i += NT) {
    const uint64_t key = top[i];
    const bool in = key != 0 && key >= bound;
    const uint64_t mask = __ballot(in);
    if (!mask) continue;
    const int first = __ffsll((unsigned long long)mask) - 1;
    uint32_t base = 0;
    if (lane == first) base = atomicAdd(&L.count, (uint32_t)__popcll(mask));
    base = __shfl(base, first);
    if (in) keys[base + __popcll(mask & ((1ull << lane) - 1))] = key;
  }
  __syncthreads();
  const int m = (int)L.count;
  for (int i = tid; i < m; i += NT) {
    const uint64_t key = keys[i];
    int r = 0;
    for (int j = 0; j < m; ++j) r += keys[j] > key;
    if (r < a.k) {
      a.top_ids[row * a.k + r] = (int32_t)(0xFFFFFFFFu - (uint32_t)key);
      a.top_logprobs[row * a.k + r] = logp(from_ord((uint32_t)(key >> 32)));
    }
  }
}

// ------------------------------------------------------------- backward
struct BwdArgs {
  const void* logits;
  void* grad;
  int64_t ld, ld_grad;
  int rows, V, np, n_ids;
  float inv_temp;
  const int32_t* ids;
  const float* g_logp;
  const float* lse;
  const float* entropy;
  const float* g_ent;
};

template <typename T>
__device__ __forceinline__ void store_chunk(T* row, int e, int V, const float* v) {
  using E = Elems<T>;
  if (e + E::n <= V) {
    u32x4 o;
    if constexpr (sizeof(T) == 2) {
      typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)v[2 * j], (__bf16)v[2 * j + 1]});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __float_as_uint(v[j]);
    }
    *reinterpret_cast<u32x4_any*>(row + e) = o;
    return;
  }
#pragma unroll
  for (int j = 0; j < E::n; ++j)
    if (e + j < V) {
      if constexpr (sizeof(T) == 2) row[e + j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
      else row[e + j] = v[j];
    }
}

// One workgroup per piece of a row, 8 KB (two chunks a thread: a workgroup
// reads all of its piece before it writes, and the shorter it is the better the
// two mix over the chip: 4096 x 128256 bf16 350 us, 6.0 TB/s read and written;
// with eight, four and one chunks a thread 404, 402 and 445 where it took 362).
// dx = (sum_j g_j [v = id_j] - p (G + g_ent (logp + H))) / temperature, G = sum
// g_j. grad may be logits: a workgroup reads its piece before it writes it, and
// the given tokens' logits before any of it is written.
//
// p comes from the f32 lse, whose rounding is |lse| 2^-24 of it: at most 2^-12
// below kLseMax. At 1e8 log V is lost and past 3e38 lse is infinite; rows from
// kLseMax on are one workgroup's, which forms their maximum and sum again
// (4096 x 128256 bf16, every row such: 1460 us against 350; 4 rows 57 against 9).
constexpr float kLseMax = 4096.f;
constexpr int kBwdChunks = 2;
template <typename T>
constexpr int kBwdPiece = kThreads * kBwdChunks * Elems<T>::n;

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(const BwdArgs a) {
  using E = Elems<T>;
  const int tid = threadIdx.x;
  const uint32_t at = piece_index(blockIdx.x, gridDim.x);
  const int64_t row = at / a.np;
  const int piece = (int)(at % a.np), e0 = piece * kBwdPiece<T>;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  T* out = static_cast<T*>(a.grad) + row * a.ld_grad;
  const int32_t* ids = a.ids + row * a.n_ids;
  const float* gl = a.g_logp + row * a.n_ids;
  float G = 0.f;
  bool any = false;  // an upstream gradient that is not zero
  for (int j = 0; j < a.n_ids; ++j) {
    const int id = ids[j];
    if (id < 0) continue;
    G += id < a.V ? gl[j] : NAN;
    any = any || id >= a.V || !(gl[j] == 0.f);
  }
  const float gh = a.g_ent ? a.g_ent[row] : 0.f;
  any = any || !(gh == 0.f);
  const float lse = a.lse[row], H = a.g_ent ? a.entropy[row] : 0.f;
  auto zeros = [&](int from, int to) {
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int e = from + tid * E::n; e < to; e += kThreads * E::n) store_chunk(out, e, a.V, z);
  };
  if (!any) {  // nothing flows: zeros, whatever the logits hold
    zeros(e0, min(a.V, e0 + kBwdPiece<T>));
    return;
  }
  // log p in, without the given tokens' own terms
  auto base = [&](float d) {
    d = d < -1e4f ? -1e4f : d;  // p = 0 there: no 0 * inf; NaN stays
    return -__builtin_amdgcn_exp2f(d * kLog2e) * fmaf(gh, d + H, G);
  };
  // thread j: the j-th given token where it lies in [from, to) and has not been
  // given before, and its gradient
  int mine = -1;
  float mine_g = 0.f;
  auto given = [&](int from, int to, auto logp) {
    if (tid < a.n_ids) {
      const int id = ids[tid];
      if (id >= from && id < to) {
        mine = id;
        float g = 0.f;
        for (int j = 0; j < a.n_ids; ++j)
          if (ids[j] == id) {
            if (j < tid) mine = -1;
            g += gl[j];
          }
        mine_g = (base(logp(value_of(x[id]))) + g) * a.inv_temp;
      }
    }
    if (a.n_ids) __syncthreads();
  };
  auto put_given = [&]() {
    if (!a.n_ids) return;
    __syncthreads();
    if (mine >= 0) {
      if constexpr (sizeof(T) == 2) out[mine] = __builtin_bit_cast(uint16_t, (__bf16)mine_g);
      else out[mine] = mine_g;
    }
  };
  if (!(fabsf(lse) < kLseMax) && lse == lse) {
    // The first piece's workgroup alone, as it reads all of the row before it
    // writes any: log p from the row's own maximum and sum.
    if (piece) return;
    __shared__ float s_m[kWaves];
    __shared__ double s_s[kWaves];
    float m = -INFINITY;
#pragma unroll 1
    for (int e = tid * E::n; e < a.V; e += kThreads * E::n) {
      const u32x4 c = load_chunk(x, e, a.V);
#pragma unroll
      for (int j = 0; j < E::n; ++j) m = fmaxf(m, E::get(c, j));
    }
    m = wave_max(m);
    if ((tid & 63) == 0) s_m[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    if (m == -INFINITY) {  // nothing is allowed
      zeros(0, a.V);
      return;
    }
    double sum = 0.0;
#pragma unroll 1
    for (int e = tid * E::n; e < a.V; e += kThreads * E::n) {
      const u32x4 c = load_chunk(x, e, a.V);
#pragma unroll
      for (int j = 0; j < E::n; ++j) sum += __builtin_amdgcn_exp2f((E::get(c, j) - m) * a.inv_temp * kLog2e);
    }
    sum = wave_sum64(sum);
    if ((tid & 63) == 0) s_s[tid >> 6] = sum;
    __syncthreads();
    const float log_sum = (float)(log2(s_s[0] + s_s[1] + s_s[2] + s_s[3]) * kLn2);
    auto logp = [&](float v) { return fmaf(v - m, a.inv_temp, -log_sum); };
    given(0, a.V, logp);
#pragma unroll 1
    for (int e = tid * E::n; e < a.V; e += kThreads * E::n) {
      const u32x4 c = load_chunk(x, e, a.V);
      float v[E::n];
#pragma unroll
      for (int j = 0; j < E::n; ++j) v[j] = base(logp(E::get(c, j))) * a.inv_temp;
      store_chunk(out, e, a.V, v);
    }
    put_given();
    return;
  }
  u32x4 ch[kBwdChunks];
#pragma unroll
  for (int q = 0; q < kBwdChunks; ++q) ch[q] = load_chunk(x, e0 + (q * kThreads + tid) * E::n, a.V);
  auto logp = [&](float v) { return fmaf(v, a.inv_temp, -lse); };
  given(e0, min(a.V, e0 + kBwdPiece<T>), logp);
#pragma unroll
  for (int q = 0; q < kBwdChunks; ++q) {
    const int e = e0 + (q * kThreads + tid) * E::n;
    float v[E::n];
#pragma unroll
    for (int j = 0; j < E::n; ++j) v[j] = base(logp(E::get(ch[q], j))) * a.inv_temp;
    if (e < a.V) store_chunk(out, e, a.V, v);
  }
  put_given();
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
int pieces(int V, int dtype) {
  const int p = dtype == GLT_DTYPE_BF16 ? kPiece<uint16_t> : kPiece<float>;
  return (V + p - 1) / p;
}
size_t parts_bytes(int rows, int V, int dtype) { return round256((size_t)rows * pieces(V, dtype) * kWaves * sizeof(Part)); }

int bwd_pieces(int V, int dtype) {
  const int p = dtype == GLT_DTYPE_BF16 ? kBwdPiece<uint16_t> : kBwdPiece<float>;
  return (V + p - 1) / p;
}

glt_status check_rows(const char* who, int32_t dtype, int64_t ld, int32_t rows, int32_t V, float temperature, int32_t n_ids) {
  GLT_CHECK(dtype == GLT_DTYPE_BF16 || dtype == GLT_DTYPE_F32, GLT_ERR_DTYPE, "%s: dtype %d", who, dtype);
  GLT_CHECK(rows >= 0 && V > 0 && ld >= V, GLT_ERR_SHAPE, "%s: rows=%d V=%d ld=%lld", who, rows, V, (long long)ld);
  GLT_CHECK(V <= kMaxV, GLT_ERR_UNSUPPORTED, "%s: V=%d (at most %d)", who, V, kMaxV);
  GLT_CHECK(n_ids >= 0 && n_ids <= kMaxIds, GLT_ERR_UNSUPPORTED, "%s: %d given tokens a row (at most %d)", who, n_ids, kMaxIds);
  // 1 / temperature and log2(e) / temperature are finite and not zero
  GLT_CHECK(temperature > 1e-30f && temperature < 1e30f, GLT_ERR_INVALID_ARG, "%s: temperature %g", who, (double)temperature);
  // a launch holds less than 2^32 threads
  GLT_CHECK((int64_t)rows * pieces(V, dtype) < (1ll << 32) / kThreads, GLT_ERR_SHAPE, "%s: rows=%d V=%d", who, rows, V);
  return GLT_OK;
}

template <typename T>
glt_status launch_fwd(const FwdArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * a.np));
  if (a.k > 0) GLT_LAUNCH("logprobs", (logprobs_piece_kernel<T, true>), grid, dim3(kThreads), 0, st, a);
  else GLT_LAUNCH("logprobs", (logprobs_piece_kernel<T, false>), grid, dim3(kThreads), 0, st, a);
  GLT_LAUNCH_CHECK("logprobs");
  const int nk = a.np * a.k;
  if (nk * 8 > kLdsFree) {
    // the dynamic-LDS limit is a per-device attribute of the kernel
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    GLT_TRY_HIP(hipGetDevice(&dev));
    GLT_CHECK(dev >= 0 && dev < 64, GLT_ERR_HIP, "glt_token_logprobs: device index %d out of range", dev);
    if (!attr_set[dev].load(std::memory_order_acquire)) {
      GLT_TRY_HIP(hipFuncSetAttribute((const void*)logprobs_row_kernel<T, kThreads>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                      kMaxV / kPiece<T> * kMaxTop * 8));
      attr_set[dev].store(true, std::memory_order_release);
    }
  }
  if (nk <= 64)
    GLT_LAUNCH("logprobs_row", (logprobs_row_kernel<T, 64>), dim3((unsigned)a.rows), dim3(64), (size_t)nk * 8, st, a);
  else
    GLT_LAUNCH("logprobs_row", (logprobs_row_kernel<T, kThreads>), dim3((unsigned)a.rows), dim3(kThreads), (size_t)nk * 8, st, a);
  GLT_LAUNCH_CHECK("logprobs_row");
  return GLT_OK;
}

}  // namespace

}  // namespace glt

using namespace glt;

extern "C" {

size_t glt_token_logprobs_workspace_size(int32_t rows, int32_t V, int32_t dtype, int32_t top_k) {
  if (rows <= 0 || V <= 0 || top_k < 0 || (dtype != GLT_DTYPE_BF16 && dtype != GLT_DTYPE_F32)) return 256;
  return parts_bytes(rows, V, dtype) + round256((size_t)rows * pieces(V, dtype) * top_k * 8);
}

glt_status glt_token_logprobs(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t V, float temperature,
                              const int32_t* ids, int32_t n_ids, int32_t top_k, float* logprobs, float* entropy,
                              float* lse, int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const char* who = "glt_token_logprobs";
  const glt_status s = check_rows(who, dtype, ld, rows, V, temperature, n_ids);
  if (s != GLT_OK) return s;
  GLT_CHECK(top_k >= 0 && top_k <= kMaxTop && top_k <= V, GLT_ERR_UNSUPPORTED, "%s: top_k %d (at most %d, and V=%d)", who,
            top_k, kMaxTop, V);
  if (rows == 0) return GLT_OK;
  GLT_CHECK(logits && (n_ids == 0 || (ids && logprobs)) && (top_k == 0 || (top_ids && top_logprobs)),
            GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  const int es = dtype == GLT_DTYPE_BF16 ? 2 : 4;
  GLT_CHECK((uintptr_t)logits % es == 0 && ((uintptr_t)ids | (uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)lse |
                                            (uintptr_t)top_ids | (uintptr_t)top_logprobs) % 4 == 0,
            GLT_ERR_ALIGNMENT, "%s: pointers must be aligned to their elements", who);
  const size_t need = glt_token_logprobs_workspace_size(rows, V, dtype, top_k);
  GLT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, GLT_ERR_WORKSPACE,
            "%s: needs %zu workspace bytes, 256-byte aligned", who, need);
  FwdArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.rows = rows; a.V = V; a.np = pieces(V, dtype); a.n_ids = n_ids; a.k = top_k;
  a.c = (float)(1.4426950408889634074 / (double)temperature);
  a.ids = ids;
  a.parts = static_cast<Part*>(workspace);
  a.top = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + parts_bytes(rows, V, dtype));
  a.logprobs = logprobs; a.entropy = entropy; a.lse = lse; a.top_ids = top_ids; a.top_logprobs = top_logprobs;
  return dtype == GLT_DTYPE_BF16 ? launch_fwd<uint16_t>(a, as_stream(stream)) : launch_fwd<float>(a, as_stream(stream));
}

glt_status glt_token_logprobs_bwd(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t V,
                                  float temperature, const int32_t* ids, int32_t n_ids, const float* grad_logprobs,
                                  const float* lse, const float* entropy, const float* grad_entropy, void* grad,
                                  int64_t ld_grad, void* stream) {
  const char* who = "glt_token_logprobs_bwd";
  const glt_status s = check_rows(who, dtype, ld, rows, V, temperature, n_ids);
  if (s != GLT_OK) return s;
  GLT_CHECK(ld_grad >= V, GLT_ERR_SHAPE, "%s: ld_grad=%lld V=%d", who, (long long)ld_grad, V);
  GLT_CHECK((int64_t)rows * bwd_pieces(V, dtype) < (1ll << 32) / kThreads, GLT_ERR_SHAPE,
            "%s: rows=%d V=%d are more workgroups than a launch holds", who, rows, V);
  if (rows == 0) return GLT_OK;
  GLT_CHECK(logits && grad && lse && (n_ids == 0 || (ids && grad_logprobs)) && (!grad_entropy || entropy),
            GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(grad != logits || ld_grad == ld, GLT_ERR_SHAPE, "%s: in place with strides %lld and %lld", who, (long long)ld,
            (long long)ld_grad);
  const int es = dtype == GLT_DTYPE_BF16 ? 2 : 4;
  GLT_CHECK(((uintptr_t)logits | (uintptr_t)grad) % es == 0 &&
                ((uintptr_t)ids | (uintptr_t)grad_logprobs | (uintptr_t)lse | (uintptr_t)entropy | (uintptr_t)grad_entropy) % 4 == 0,
            GLT_ERR_ALIGNMENT, "%s: pointers must be aligned to their elements", who);
  // a workgroup writes its piece while others still read theirs and their row's values
  const ByteRows to{grad, rows, (int64_t)V * es, ld_grad * es};
  GLT_CHECK(grad == logits || !overlap(to, {logits, rows, (int64_t)V * es, ld * es}), GLT_ERR_INVALID_ARG,
            "%s: grad overlaps the logits without being them", who);
  for (const void* x : {static_cast<const void*>(lse), static_cast<const void*>(entropy), static_cast<const void*>(grad_entropy)})
    GLT_CHECK(!x || !overlap(to, dense_bytes(x, (int64_t)rows * 4)), GLT_ERR_INVALID_ARG, "%s: grad overlaps an input", who);
  for (const void* x : {static_cast<const void*>(ids), static_cast<const void*>(grad_logprobs)})
    GLT_CHECK(n_ids == 0 || !overlap(to, dense_bytes(x, (int64_t)rows * n_ids * 4)), GLT_ERR_INVALID_ARG,
              "%s: grad overlaps an input", who);
  const BwdArgs a{logits, grad, ld, ld_grad, rows, V, bwd_pieces(V, dtype), n_ids, (float)(1.0 / (double)temperature), ids,
                  grad_logprobs, lse, entropy, grad_entropy};
  const dim3 grid((unsigned)(rows * a.np));
  if (dtype == GLT_DTYPE_BF16)
    GLT_LAUNCH("logprobs_bwd", logprobs_bwd_kernel<uint16_t>, grid, dim3(kThreads), 0, as_stream(stream), a);
  else
    GLT_LAUNCH("logprobs_bwd", logprobs_bwd_kernel<float>, grid, dim3(kThreads), 0, as_stream(stream), a);
  GLT_LAUNCH_CHECK("logprobs_bwd");
  return GLT_OK;
}

}  // extern "C"

// Attention of new tokens over the 8-bit cache of keys and values, for gfx950.
//
// A key j of a segment (a sequence's own tokens, or a prefix that a group of
// sequences shares) is seen by a row at position p if
//   j <= p  and  (no window  or  j > p - window  or  j < sinks).
// The codes are whole numbers of 7 bits and a sign: bf16 holds them exactly, so
//   s = (q . code_k) step_k scale,   o += (p step_v) . code_v
// need one rounding, of p step_v, and no value of k or v is formed.
//
// Everything that the new tokens have to read is a list of tiles of work, dealt out in
// equal runs (Dealt below): whatever the lengths, each wavefront or workgroup gets its
// share. Where a run ends inside of a segment its rows come in pieces: a piece's output,
// maximum and sum go into the workspace, and a last kernel joins each row's pieces in
// order. Few rows a segment (new tokens x query heads of a kv head: few_rows) or many
// (many_rows); the kinds of a call's own tokens and prefixes run in one launch. Short
// caches need one launch in all (kv8_whole_kernel).
//
// Masks are formed with & and |: from && and || the compiler (ROCm 7.2) made branches of
// which one lost a masked score.
//
// p is off by the rounding of p step_v, out by that and its own: 1.9 to 2.2 * 10^-3 in the
// 2-norm, of which its own is 1.6.
#include <algorithm>
#include <atomic>

#include "attention_dev.hpp"
#include "kv8.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

constexpr float kSlack = 8.0f;      // running-max slack (log2 units)
constexpr float kNoMax = -3.4028234663852886e38f;  // maximum of a row that has seen nothing: below every score's

// A kind of segments, [0] the sequences' own tokens, [1] prefixes.
struct Part {
  int rows;        // of a segment and head
  int workers;     // wavefronts (few rows) or workgroups (many) that the work is dealt to
  int blocks;      // workgroups of the launch
  int* first;      // tiles of work before each segment, and in all
  float* o;        // pieces' results by slot and row: 128 each
  float* m;        // maximum (log2 units) and sum
};
struct DecArgs {
  const uint8_t* cache;
  int64_t n_pages;
  glt_kv8_seqs s;
  const int32_t* ppages;
  const int32_t* plens;
  int64_t prefix_ld;
  int n_prefix_table, n_groups, gs;  // gs: sequences of a group
  int Hkv, G, W, S;
  float scale_log2;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  int64_t q_ld, o_ld;
  Part part[2];
};

__device__ __forceinline__ int prefix_len(const DecArgs& a, int b) {
  return a.n_groups ? min(max(a.plens[b / a.gs], 0), a.n_prefix_table * kPage) : 0;
}

// What the segment's rows see of it: of its first `hi` keys those from `lo` on and the
// first `sunk`; a list of n pages, ns that hold sinks and then those from c0 on.
struct Sight {
  int hi, ns, c0, n;
  __device__ __forceinline__ int page(int i) const { return i < ns ? i : c0 + i - ns; }
};
template <bool PRE>
__device__ __forceinline__ Sight sight(const DecArgs& a, int seg) {
  int hi, lo = 0, sunk = 0;
  if (PRE) {
    hi = min(max(a.plens[seg], 0), a.n_prefix_table * kPage);
    if (a.W) {
      int from = INT32_MAX;  // the earliest new token of the group
      for (int b = seg * a.gs; b < (seg + 1) * a.gs; ++b) {
        const Kv8Len n = kv8_len(a.s, b);
        if (n.fresh > 0) from = min(from, hi + n.len - n.fresh);
      }
      if (from == INT32_MAX) hi = 0;
      lo = max(from - a.W + 1, 0);
      sunk = min(a.S, hi);
    }
  } else {
    const Kv8Len n = kv8_len(a.s, seg);
    hi = n.fresh > 0 ? n.len : 0;
    if (a.W && hi) {
      lo = max(n.len - n.fresh - a.W + 1, 0);
      sunk = min(max(a.S - prefix_len(a, seg), 0), hi);
    }
  }
  Sight r;
  r.hi = hi;
  const int end = (hi + kPage - 1) / kPage;
  r.c0 = min(lo / kPage, end);
  r.ns = min((sunk + kPage - 1) / kPage, r.c0);
  r.n = r.ns + end - r.c0;
  return r;
}

// A row's sight within a segment: key j is seen if j < hi and (j >= lo or j < sunk).
struct Row {
  int hi, lo, sunk;
  int64_t q_row;  // b * T + t, and its head, for q and the outputs
  int head;
};
template <bool PRE>
__device__ __forceinline__ Row row_of(const DecArgs& a, int seg, int h, int r, int seg_hi) {
  const int per = a.s.T * a.G;
  const int b = PRE ? seg * a.gs + r / per : seg;
  const int x = PRE ? r % per : r, t = x / a.G;
  const Kv8Len n = kv8_len(a.s, b);
  const int P = prefix_len(a, b);
  Row w;
  w.q_row = (int64_t)b * a.s.T + t;
  w.head = h * a.G + x % a.G;
  const int own = n.len - n.fresh + t;  // position among its own tokens
  const bool live = t < n.fresh;
  w.hi = !live ? 0 : PRE ? seg_hi : min(own + 1, seg_hi);
  w.lo = a.W ? max((PRE ? P + own : own) - a.W + 1, 0) : 0;
  w.sunk = a.W ? max(PRE ? a.S : a.S - P, 0) : 0;
  return w;
}

template <bool PRE>
__device__ __forceinline__ int page_id(const DecArgs& a, int seg, int p) {
  return PRE ? a.ppages[seg * a.prefix_ld + p] : a.s.pages[seg * a.s.pages_ld + p];
}
// Where a page's head lies; a page outside the pool is not followed (its scores count as
// NaN).
__device__ __forceinline__ bool page_ok(const DecArgs& a, int id) { return id >= 0 && id < a.n_pages; }
__device__ __forceinline__ const uint8_t* page_at(const DecArgs& a, int id, int h) {
  return a.cache + ((int64_t)(page_ok(a, id) ? id : 0) * a.Hkv + h) * kHeadB;
}

// Eight codes as bf16 (exact: the upper halves of their f32 values).
__device__ __forceinline__ bf16x8 codes8(uint32_t x, uint32_t y) {
  auto f = [](uint32_t w, int e) { return __float_as_uint((float)(int8_t)(w >> (8 * e))); };
  auto two = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); };
  return __builtin_bit_cast(bf16x8, u32x4{two(f(x, 0), f(x, 1)), two(f(x, 2), f(x, 3)), two(f(y, 0), f(y, 1)), two(f(y, 2), f(y, 3))});
}

__device__ __forceinline__ float quad_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_max(fmax_nc(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A finished row's lse and output: nothing seen gives -inf and zeros, NaN stays.
__device__ __forceinline__ void write_lse(const DecArgs& a, const Row& w, float m, float l) {
  const int64_t b = w.q_row / a.s.T, t = w.q_row - b * a.s.T;
  a.lse[(b * a.Hkv * a.G + w.head) * a.s.T + t] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}
// N groups of four channels from 4 lane on, STEP apart, of this lane
template <int STEP, int N>
__device__ __forceinline__ void write_row(const DecArgs& a, const Row& w, const f32x4* o, float m, float l, int lane) {
  const float f = l == 0.f ? 0.f : 1.0f / l;
  uint16_t* to = a.out + w.q_row * a.o_ld + (int64_t)w.head * kKv8Hd + 4 * lane;
#pragma unroll
  for (int i = 0; i < N; ++i)
    *reinterpret_cast<u32x2a*>(to + STEP * i) = u32x2a{pack2_rne(o[i][0] * f, o[i][1] * f), pack2_rne(o[i][2] * f, o[i][3] * f)};
  if (lane == 0) write_lse(a, w, m, l);
}

// ---------------------------------------------------------------- dealing
constexpr int kManyRows = 256;  // rows of a workgroup of many_rows
constexpr int kFewRows = 32;    // rows that few_rows takes

// Row blocks of a segment that hold new tokens.
template <bool PRE, bool MANY>
__device__ __forceinline__ int row_blocks(const DecArgs& a, int seg) {
  if (!MANY) return 1;
  return ((PRE ? a.part[1].rows : kv8_len(a.s, seg).fresh * a.G) + kManyRows - 1) / kManyRows;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Sum over this and the lanes before.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // rows of 16, shifted by 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // a row's last lane to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}

// Tiles of work (pages x row blocks) before each segment and in all, for a workgroup; its
// first one writes them for the join too. Up to 64 segments every wavefront keeps in a
// register, a lane each: no barrier, and one comparison finds a tile's segment.
template <int WAVES, bool PRE, bool MANY>
struct Dealt {
  int* lds;   // [n_seg + 1] of more than 64 segments
  int mine;   // before segment `lane`
  int n_seg, total;

  __device__ __forceinline__ Dealt(const DecArgs& a, int* at, int block) : lds(at) {
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    n_seg = PRE ? a.n_groups : a.s.B;
    auto tiles = [&](int s) { return s < n_seg ? sight<PRE>(a, s).n * row_blocks<PRE, MANY>(a, s) : 0; };
    if (n_seg <= 64) {
      const int n = tiles(lane), x = wave_scan(n);
      mine = x - n;
      total = __builtin_amdgcn_readlane(x, 63);
      if (block == 0 && wave == 0) {
        if (lane < n_seg) a.part[PRE].first[lane] = mine;
        if (lane == 0) a.part[PRE].first[n_seg] = total;
      }
      return;
    }
    __shared__ int wave_sum[WAVES];
    total = 0;
    for (int s0 = 0; s0 < n_seg; s0 += WAVES * 64) {
      const int n = tiles(s0 + tid), x = wave_scan(n);
      if (lane == 63) wave_sum[wave] = x;
      __syncthreads();
      int before = total;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += wave_sum[w];
        total += wave_sum[w];
      }
      if (s0 + tid < n_seg) lds[s0 + tid] = before + x - n;
      if (s0 + tid == n_seg - 1) lds[n_seg] = total;
      __syncthreads();
    }
    total = uni(total);
    if (block == 0)
      for (int s = tid; s <= n_seg; s += WAVES * 64) a.part[PRE].first[s] = lds[s];
  }
  __device__ __forceinline__ int first(int seg) const {
    if (n_seg > 64) return uni(lds[seg]);
    return seg < n_seg ? __builtin_amdgcn_readlane(mine, seg) : total;
  }
  // The segment that tile `pos` of a head lies in: the last one that starts at or before it.
  __device__ __forceinline__ int find(int pos) const {
    if (n_seg <= 64) return uni(__popcll(__ballot((int)(threadIdx.x & 63) < n_seg && mine <= pos)) - 1);
    int seg = 0;
    for (int end = n_seg; end - seg > 1;) {
      const int mid = (seg + end) >> 1;
      if (first(mid) <= pos) seg = mid;
      else end = mid;
    }
    return seg;
  }
};
// Tiles of a run.
template <bool MANY>
__device__ __forceinline__ int run_tiles(int all, int workers) {
  return max((all + workers - 1) / workers, MANY ? 2 : 1);
}
// Slot of a piece of a column (segment, head, row block). A worker has one piece that
// goes on with a column (its first) and one that begins a column without ending it (its
// last); where prefixes' pieces have to be joined to them, whole columns need a slot
// too: workers and columns both rise along the list.
template <bool PRE>
__device__ __forceinline__ int64_t slot_of(const DecArgs& a, int worker, int64_t column, bool begins) {
  return PRE || a.n_groups ? worker + column : 2 * (int64_t)worker + begins;
}

// -------------------------------------------------------------- few rows
// Up to 16 NB rows a segment and head: a tile is a page of a head, and the workers are
// wavefronts. A wavefront loads a page's codes with 16-byte loads straight into the operands of
//   S^T[key][row] = K . Q^T,  O^T[channel][row] += V^T . P^T
// (16 x 16 x 32), with the softmax between: no LDS, no barrier, and every code is
// converted once (1.5 vector instructions a code: a conversion to f32, of which the upper half is
// the bf16, and half a byte permutation).
//
// Bound by memory: 32 sequences of 1 to 32768 tokens, 8 kv heads (1.09 GB) in 190 us, 5.7
// TB/s (a large copy: 5.2), three wavefronts of 17 KB in flight on each SIMD; at two the same
// takes 250 with a piece for each 8 pages and a barrier behind it. The four rows of a
// kv head's query heads leave 12 of the products' 16 columns empty, which costs nothing:
// the matrix instructions run 0.07 of the time, vector ones 0.35.
//
// Lane l: row l & 15 of a block of 16, g = l >> 4. The keys of score block (beta, a) are
// numbered so that the accumulators are the second product's operand as they stand:
// element e of lane group g is key 16 g + 8 a + 4 beta + e of the page.
template <int NB>
struct Few {
  Row row[NB];
  bf16x8 qf[NB][4];
  f32x4 o[NB][8];
  float m[NB], l[NB];

  // (what depends on the lane is worked out for each run: kept, it costs registers
  // that there are not)
  template <bool PRE>
  __device__ __forceinline__ void begin(const DecArgs& a, int seg, int h, int seg_hi) {
    const int lane = (int)opaque(threadIdx.x) & 63, R = a.part[PRE].rows;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      row[nb] = row_of<PRE>(a, seg, h, min(16 * nb + (lane & 15), R - 1), seg_hi);
      const uint16_t* qp = a.q + row[nb].q_row * a.q_ld + (int64_t)row[nb].head * kKv8Hd + 16 * (lane >> 4);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        qf[nb][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qp + 64 * (s >> 1) + 8 * (s & 1)));
      m[nb] = kNoMax;
      l[nb] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[nb][i] = f32x4{};
    }
  }

  // page p of the segment, at pg
  __device__ __forceinline__ void page(const DecArgs& a, const uint8_t* pg, bool ok, int p) {
    const int lane = (int)(NB > 1 ? opaque(threadIdx.x) : threadIdx.x) & 63, r15 = lane & 15, g = lane >> 4;
    u32x4 kx[8], vx[8], kst[2], vst[2];
    const uint8_t* kp = pg + (uint32_t)((16 * (r15 >> 2) + (r15 & 3)) * kKv8Hd + 16 * g);
#pragma unroll
    for (int i = 0; i < 8; ++i)  // block (beta = i >> 2, a = (i >> 1) & 1), channels 64 (i & 1) + 16 g ..
      kx[i] = *reinterpret_cast<const u32x4*>(kp + (8 * ((i >> 1) & 1) + 4 * (i >> 2)) * kKv8Hd + 64 * (i & 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kst[i] = *reinterpret_cast<const u32x4*>(pg + (uint32_t)(kKStepOff + 32 * g + 16 * i));
      vst[i] = *reinterpret_cast<const u32x4*>(pg + (uint32_t)(kVStepOff + 32 * g + 16 * i));
    }
    auto load_v = [&](int from, int to) {
#pragma unroll
      for (int i = from; i < to; ++i) vx[i] = *reinterpret_cast<const u32x4*>(pg + (uint32_t)(kVOff + (16 * i + r15) * kPage + 16 * g));
    };
    if (NB == 1) load_v(0, 8);
    const float scale = ok ? a.scale_log2 : NAN;
    // steps of keys 16 g + i
    auto step = [](const u32x4* x, int i) {
      const uint32_t w = x[i >> 3][(i & 7) >> 1];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    };

    f32x4 s[NB][4];  // block 2 beta + a
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb][blk] = f32x4{};
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const u32x4 x = kx[2 * blk + (st >> 1)];
        const bf16x8 ka = codes8(x[2 * (st & 1)], x[2 * (st & 1) + 1]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb][blk] = mfma16(ka, qf[nb][st], s[nb][blk]);
      }
      if (NB > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (NB > 1) {  // no registers for both, nor for all of v
      __builtin_amdgcn_sched_barrier(0);
      load_v(0, 4);
    }
    bf16x8 pf[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const Row& w = row[nb];
      const int key0 = p * kPage + 16 * g;
      // every row sees the whole page, but for rows that come to nothing
      const bool whole = __all((w.hi == 0) | ((p * kPage + kPage <= w.hi) & ((p * kPage >= w.lo) | (p * kPage + kPage <= w.sunk))));
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nb][blk][e] *= step(kst, 8 * (blk & 1) + 4 * (blk >> 1) + e) * scale;
      if (!whole)
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = key0 + 8 * (blk & 1) + 4 * (blk >> 1) + e;
            const bool in = (j < w.hi) & ((j >= w.lo) | (j < w.sunk));
            s[nb][blk][e] = in ? s[nb][blk][e] : -INFINITY;
          }
      float mt = s[nb][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mt = fmax_nc(mt, s[nb][i >> 2][i & 3]);
      mt = quad_max(mt);
      // (each row's moves by itself: no other row's values touch it)
      const bool up = mt > m[nb] + kSlack;
      if (__any(up)) {
        const float m_new = up ? mt : m[nb];
        const float alpha = __builtin_amdgcn_exp2f(m[nb] - m_new);
        m[nb] = m_new;
        l[nb] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[nb][i] *= alpha;
      }
      float pv[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(s[nb][i >> 2][i & 3] - m[nb]);
        l[nb] += x;
        pv[i] = x * step(vst, 8 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3));
      }
      if (!whole)  // an unseen key's step may be anything
#pragma unroll
        for (int i = 0; i < 16; ++i) pv[i] = s[nb][i >> 2][i & 3] == -INFINITY ? 0.f : pv[i];
#pragma unroll
      for (int beta = 0; beta < 2; ++beta) {
        const float* x = pv + 8 * beta;
        pf[nb][beta] = __builtin_bit_cast(bf16x8, u32x4{pack2_rne(x[0], x[1]), pack2_rne(x[2], x[3]), pack2_rne(x[4], x[5]),
                                                        pack2_rne(x[6], x[7])});
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (NB > 1 && i == 0) load_v(4, 8);
#pragma unroll
      for (int beta = 0; beta < 2; ++beta) {
        const bf16x8 va = codes8(vx[i][2 * beta], vx[i][2 * beta + 1]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb][i] = mfma16(va, pf[nb][beta], o[nb][i]);
      }
    }
  }
};

template <int WAVES, int NB, bool PRE>
__device__ __forceinline__ void few_rows(const DecArgs& a, int* first, int block) {
  const int n_seg = PRE ? a.n_groups : a.s.B, R = a.part[PRE].rows;
  const Dealt<WAVES, PRE, false> deal(a, first, block);
  const int total = deal.total;
  const int worker = block * WAVES + uni(threadIdx.x >> 6), all = total * a.Hkv;
  const int run = run_tiles<false>(all, a.part[PRE].workers);
  int at = worker * run;  // workers * run stays below all + workers
  const int stop = min(at + run, all);
  while (at < stop) {
    const int h = at / total, pos = at - h * total, seg = deal.find(pos);
    const int i0 = pos - deal.first(seg), n = deal.first(seg + 1) - deal.first(seg), i1 = min(n, i0 + stop - at);
    at += i1 - i0;
    const Sight si = sight<PRE>(a, seg);
    // lane x: the id of the run's page i + x, 64 at a time, the first ones on their way
    // while the rows are looked up
    auto ids_from = [&](int i) {
      const int x = i + (int)(threadIdx.x & 63);
      return x < i1 ? page_id<PRE>(a, seg, a.W ? si.page(x) : x) : 0;
    };
    int ids = ids_from(i0);
    Few<NB> f;
    f.template begin<PRE>(a, seg, h, si.hi);
    for (int i = i0; i < i1; ++i) {
      const int x = (i - i0) & 63;
      if (x == 0 && i > i0) ids = ids_from(i);
      const int id = __builtin_amdgcn_readlane(ids, x);
      f.page(a, page_at(a, id, h), page_ok(a, id), a.W ? si.page(i) : i);
    }
    const int l2 = (int)opaque(threadIdx.x) & 63, c15 = l2 & 15, cg = l2 >> 4;
    const bool done = !PRE && !a.n_groups && i1 - i0 == n;  // the rows' only piece
    const int64_t slot = slot_of<PRE>(a, worker, (int64_t)h * n_seg + seg, i0 == 0);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float l = quad_sum(f.l[nb]);
      const int r = 16 * nb + c15;
      if (r >= R) continue;
      if (done) {
        const Row w = row_of<PRE>(a, seg, h, r, si.hi);
        if (w.hi) write_row<16, 8>(a, w, f.o[nb], f.m[nb], l, cg);  // (else the join does)
        continue;
      }
      float* to = a.part[PRE].o + (slot * R + r) * kKv8Hd + 4 * cg;
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<f32x4*>(to + 16 * i) = f.o[nb][i];
      if (cg == 0) {
        a.part[PRE].m[2 * (slot * R + r)] = f.m[nb];
        a.part[PRE].m[2 * (slot * R + r) + 1] = l;
      }
    }
  }
}

// One workgroup a sequence and head, its pages dealt to WAVES wavefronts and joined in
// LDS: where the pages are few this one launch ends sooner than pieces and their join. us
// of one against the other, 32 query and 8 kv heads: 1 sequence of 1500 tokens 14.2, 15.9; 8 of
// up to 1600 14.5, 16.1; 8 of 2000 19.0, 16.3; 48 with a window of 1024 24.7, 30.0; 64 of
// 2000 44.7, 51.2; 200 of up to 1800 84, 103; 64 of up to 4000 77, 52.
template <int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 3) kv8_whole_kernel(const DecArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int R = a.part[0].rows, wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int h = blockIdx.x % a.Hkv, seg = blockIdx.x / a.Hkv;
  const Sight si = sight<false>(a, seg);
  // lane x: the id of page wave + WAVES x (of at most 32)
  const int own = wave + WAVES * lane, ids = own < si.n ? page_id<false>(a, seg, si.page(own)) : 0;
  Few<1> f;
  f.template begin<false>(a, seg, h, si.hi);
  for (int i = wave, x = 0; i < si.n; i += WAVES, ++x) {
    const int id = __builtin_amdgcn_readlane(ids, x);
    f.page(a, page_at(a, id, h), page_ok(a, id), si.page(i));
  }
  float* const ml = reinterpret_cast<float*>(smem);             // [WAVES][2][R]
  f32x4* const ov = reinterpret_cast<f32x4*>(smem + WAVES * 128);  // [WAVES][R][32]
  const float l = quad_sum(f.l[0]);
  const int r15 = lane & 15, g = lane >> 4;
  if (r15 < R) {
    if (g == 0) {
      ml[wave * 32 + r15] = f.m[0];
      ml[wave * 32 + 16 + r15] = l;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ov[(wave * R + r15) * 32 + 4 * i + g] = f.o[0][i];
  }
  __syncthreads();
  for (int x = threadIdx.x; x < R * 32; x += WAVES * 64) {
    const int r = x >> 5;
    float M = ml[r], L = 0.f;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) M = fmax_nc(M, ml[w * 32 + r]);
    f32x4 acc{};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float c = __builtin_amdgcn_exp2f(ml[w * 32 + r] - M);
      L += ml[w * 32 + 16 + r] * c;
      acc += ov[(w * R + r) * 32 + (x & 31)] * c;
    }
    const Row w = row_of<false>(a, seg, h, r, si.hi);
    if (w.hi == 0) {  // padding: zeros and -inf
      acc = f32x4{};
      L = 0.f;
    }
    write_row<4, 1>(a, w, &acc, M, L, x & 31);
  }
}

// ------------------------------------------------------------- many rows
// A column is 256 rows of a segment and head, a tile one of its pages, and the workers are
// workgroups of eight wavefronts; a wavefront owns 32 rows as in attention for training
// (attention_train.hip), two share a SIMD. Converted codes lie in LDS in the order in which the
// products' operands are read (1 KB of 64 lanes each, padded so that the writes spread
// over the banks).
//
// A tile costs a wavefront as much vector arithmetic (the softmax, the codes'
// conversion) as matrix products, and one depends on the other. So the two
// wavefronts of a SIMD alternate: between two barriers one runs its products
//   M(j): o += V(j - 1) . P(j - 1)^T,  S(j) = K(j) . Q^T
// while the other turns S(j - 1) into P(j - 1) and converts its half of the next
// operands, and then they change places. The first four wavefronts (turn 0) are a phase
// ahead of the others: in phases 2 j and 2 j + 1 M(j) runs and K(j + 1), V(j) are written,
// so that two buffers of each are enough; the steps of four tiles are kept.
//
// 512 new tokens over 8704, 32 query and 8 kv heads: 95 us, 0.74 * 10^15 operations a second;
// 2048 over 8704 292 us, 0.88. Matrix instructions run 0.32 of the time and vector ones
// 0.43: a SIMD overlaps them only in part (alone the products take 0.4 of the time, the softmax
// 0.5, the conversion 0.1 and waiting for it 0.2). us at 512 and 2048 tokens, and of a prefix of
// 16384 under 64 sequences, with the join, all before operands were read ahead: like this
// 118, 325, 58; two workgroups of four wavefronts a CU, each with its own converted pages,
// 125, 377, 56; both turns at once 135, 428; conversion between the products 130, 365, 60;
// loads a phase earlier 130, 374, 62; pages brought to L2 ahead 120, 323, 59; without raised
// priority 125, 370.
//
// With a window a row block walks the pages that hold sinks and those of its own window: 4096 new
// tokens over 8192, window 128 53 us, with 4 sinks 59.
constexpr int kManyWaves = 8;
constexpr int kKFrag = 1040, kVFrag = 1056;           // bytes of an operand of 64 lanes
constexpr int kKTile = 16 * kKFrag, kVTile = 16 * kVFrag;
constexpr int kVAt = 2 * kKTile, kStepAt = kVAt + 2 * kVTile;
constexpr int kManyLds = kStepAt + 4 * 2 * kPage * 4;  // f32 steps of k (times scale) and v: 69,120 bytes

template <bool PRE>
__device__ __forceinline__ void many_rows(const DecArgs& a, char* smem, int block) {
  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, lh = lane >> 5, wave = uni(tid >> 6), turn = wave >> 2;
  const int n_seg = PRE ? a.n_groups : a.s.B, R = a.part[PRE].rows, all_rb = (R + kManyRows - 1) / kManyRows;
  const Dealt<kManyWaves, PRE, true> deal(a, reinterpret_cast<int*>(smem + kManyLds), block);
  const int total = deal.total, all = total * a.Hkv;
  const int run = run_tiles<true>(all, a.part[PRE].workers);
  lds_char* const lds = (lds_char*)smem;
  int at = block * run;
  const int stop = min(at + run, all);
  while (at < stop) {
    const int h = at / total, pos = at - h * total, seg = deal.find(pos);
    const int nrb = uni(row_blocks<PRE, true>(a, seg)), n = (deal.first(seg + 1) - deal.first(seg)) / nrb;
    const int rem = pos - deal.first(seg), rb = rem / n, i0 = rem - rb * n, i1 = min(n, i0 + stop - at);
    at += i1 - i0;
    const Sight si = sight<PRE>(a, seg);
    // Of the list, what the block's rows see: the first `sunk` pages, which hold sinks, and
    // those from the first row's window on, to the last row's own key. (Of a prefix the list as it is.)
    int sunk = si.ns, from = si.ns, to = n;
    if (!PRE) {
      const Kv8Len ln = kv8_len(a.s, seg);
      const int t0 = rb * kManyRows / a.G, t1 = min((rb * kManyRows + kManyRows - 1) / a.G, ln.fresh - 1);
      const int p1 = (ln.len - ln.fresh + t1) / kPage + 1;  // pages that hold keys up to t1's
      to = si.ns + max(p1 - si.c0, 0);
      if (a.W) {
        from = si.ns + max(max(ln.len - ln.fresh + t0 - a.W + 1, 0) / kPage - si.c0, 0);
        sunk = (min(max(a.S - prefix_len(a, seg), 0), si.hi) + kPage - 1) / kPage;  // (ns, or past where the window starts)
      }
    }
    // the piece's part of both; where sinks lie the list's entries are the pages
    const int head = uni(max(min(min(sunk, to), i1) - i0, 0)), rest = uni(max(max(from, i0), i0 + head));
    const int tiles = uni(head + max(min(to, i1) - rest, 0)), tail = uni(si.c0 - si.ns + rest - head);
    auto page_of = [&](int j) { return a.W ? j + (j < head ? i0 : tail) : i0 + j; };
    // lane x: the id of tile x, 64 at a time, the first ones on their way while the rows are looked up
    auto ids_from = [&](int j) { return j + lane < tiles ? page_id<PRE>(a, seg, page_of(j + lane)) : 0; };
    int ids = ids_from(0);
    Row w = row_of<PRE>(a, seg, h, min(rb * kManyRows + 32 * wave + lq, R - 1), si.hi);
    if (rb * kManyRows + 32 * wave + lq >= R) w.hi = 0;
    const bool works = __any(w.hi > 0);

    bf16x8 qf[8];
    load_rows(qf, a.q + w.q_row * a.q_ld + (int64_t)w.head * kKv8Hd, true, lh);
    f32x16 o[4], s[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f32x16{};
    u32x4 pw[4];
    float m_run = kNoMax, l_run = 0.f;

    auto id_of = [&](int j) {
      if ((j & 63) == 0 && j > 0) ids = ids_from(j);
      return __builtin_amdgcn_readlane(ids, j & 63);
    };
    // this thread's 16 codes of each tile: token q >> 3, channels 16 (q & 7) .., or
    // channel q >> 2 and 16 tokens
    const uint32_t q = tid;
    u32x4 kx, vx;
    uint32_t st = 0;
    float scale = 0.f;
    const uint8_t* pg = nullptr;  // of the tile whose v is next
    auto fetch_k = [&](int j) {
      const int id = id_of(j);
      pg = page_at(a, id, h);
      kx = *reinterpret_cast<const u32x4*>(pg + 16 * q);
      // (every thread: a branch around a load waits for all of them)
      st = *reinterpret_cast<const uint16_t*>(pg + kKStepOff + 2 * (q & 127));
      scale = page_ok(a, id) ? a.scale_log2 : NAN;
    };
    auto stage_k = [&](int j) {
      const int key = q >> 3, c = q & 7;
      lds_char* x = lds + (j & 1) * kKTile + ((key >> 5) * 8 + c) * kKFrag + (key & 31) * 16;
      *(lds_bf16x8*)x = codes8(kx[0], kx[1]);
      *(lds_bf16x8*)(x + 512) = codes8(kx[2], kx[3]);
      // the second half's threads write the steps
      const float f = __uint_as_float(st << 16);
      if (q >= 256 && q < 384)
        *(__attribute__((address_space(3))) float*)(lds + kStepAt + (j & 3) * 2 * kPage * 4 + 4 * (q & 127)) =
            (q & 127) < kPage ? f * scale : f;
    };
    // What is written beside M(j): K(j + 1) and V(j). (Past the end the last page once
    // more, into buffers that nothing reads then: branches around the loads cost more.)
    auto fetch = [&](int j) {
      vx = *reinterpret_cast<const u32x4*>(pg + kVOff + 16 * q);
      fetch_k(min(j + 1, tiles - 1));
    };
    auto stage = [&](int j) {
      const int d = q >> 2, s2 = q & 3;
      lds_char* x = lds + kVAt + (j & 1) * kVTile + ((d >> 5) * 4 + s2) * kVFrag + (d & 31) * 16;
      *(lds_bf16x8*)x = codes8(vx[0], vx[1]);
      *(lds_bf16x8*)(x + 512) = codes8(vx[2], vx[3]);
      stage_k(j + 1);
    };

    auto values = [&](int j) {  // o += V(j) . P^T
      const lds_char* vr = lds + kVAt + (j & 1) * kVTile + lane * 16;
      constexpr int kAhead = 4;
      bf16x8 va[kAhead];
      auto get = [&](int i) { return *(const lds_bf16x8*)(vr + ((i & 3) * 4 + (i >> 2)) * kVFrag); };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) va[i] = get(i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i & 3] = mfma(va[i % kAhead], __builtin_bit_cast(bf16x8, pw[i >> 2]), o[i & 3]);
        if (i + kAhead < 16) va[i % kAhead] = get(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // Steps of keys 32 kb + 8 i + 4 lh + e of a tile (k's times scale, or v's), read well
    // before they are used (v's by halves: there are no registers for all of them).
    f32x4 f[8];
    auto steps = [&](int j, int v, int kb) {
      const lds_char* sp = lds + kStepAt + (2 * (j & 3) + v) * kPage * 4 + 16 * lh;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * kb + i] = *(const lds_f32x4*)(sp + 128 * kb + 32 * i);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto scores = [&](int j) {
      const lds_char* kr = lds + (j & 1) * kKTile + lane * 16;
      constexpr int kAhead = 4;
      bf16x8 ka[kAhead];
      auto get = [&](int i) { return *(const lds_bf16x8*)(kr + ((i & 1) * 8 + (i >> 1)) * kKFrag); };
      s[0] = s[1] = f32x16{};
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ka[i] = get(i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i & 1] = mfma(ka[i % kAhead], qf[i >> 1], s[i & 1]);
        if (i + kAhead < 16) ka[i % kAhead] = get(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      steps(j, 0, 0);
      steps(j, 0, 1);
    };
    auto softmax = [&](int j) {
      const int key0 = page_of(j) * kPage;
      // Scores relative to the maximum so far, in one instruction each (to 0 before a row
      // has seen anything: its maximum then moves whatever it is).
      const bool unset = m_run == kNoMax;
      const float base = unset ? 0.f : m_run;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = __builtin_fmaf(s[kb][e], f[4 * kb + (e >> 2)][e & 3], -base);
      steps(j, 1, 0);
      const bool whole = __all((w.hi == 0) | ((key0 + kPage <= w.hi) & ((key0 >= w.lo) | (key0 + kPage <= w.sunk))));
      auto in = [&](int i) {  // whether the row sees key i + 4 lh of the page
        const int at = key0 + 4 * lh;
        return (i < w.hi - at) & ((i >= w.lo - at) | (i < w.sunk - at));
      };
      if (!whole)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[kb][e] = in(32 * kb + 8 * (e >> 2) + (e & 3)) ? s[kb][e] : -INFINITY;
          }
      float m2[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        m2[kb] = s[kb][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) m2[kb] = fmax_nc(m2[kb], s[kb][e]);
      }
      const float mt = pair_max(fmax_nc(m2[0], m2[1]));
      const bool up = mt > (unset ? -INFINITY : kSlack);
      if (__any(up)) {  // each row's moves by itself
        const float m_new = up ? base + mt : m_run;
        // As the new maximum is rounded, unless that puts it more than 1 off (scores past
        // 2^24): the largest probability would leave f32 or vanish.
        float by = m_new - base;
        by = !up ? 0.f : __builtin_fabsf(by - mt) > 1.f ? mt : by;
        const float alpha = unset ? 1.f : __builtin_amdgcn_exp2f(-by);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] -= by;
      }
      float ls[2] = {l_run, 0.f};
      auto probs = [&](bool masked) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          if (kb == 0) steps(j, 1, 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = __builtin_amdgcn_exp2f(s[kb][4 * i + e]);
              ls[kb] += y;
              x[e] = y * (!masked || in(32 * kb + 8 * i + e) ? f[4 * kb + i][e] : 0.f);  // an unseen key's step may be anything
            }
            pw[2 * kb + (i >> 1)][2 * (i & 1)] = pack2_rne(x[0], x[1]);
            pw[2 * kb + (i >> 1)][2 * (i & 1) + 1] = pack2_rne(x[2], x[3]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      if (whole) probs(false);
      else probs(true);
      l_run = ls[0] + ls[1];
    };

    // (the run before: its last phase reads V and the turns' barriers match, so nothing that
    // is written before the next barrier is still read)
    if (tiles > 0) {
      fetch_k(0);
      stage_k(0);
      if (turn) fetch(0);
      __builtin_amdgcn_s_waitcnt(vmcnt_enc(0));  // q too: no product has to wait for a page
      phase_barrier();
      if (turn) {
        stage(0);
        phase_barrier();
      }
      fetch(turn);
      if (works) {
        scores(0);
        for (int j = 0; j < tiles; ++j) {
          phase_barrier();
          softmax(j);
          stage(j + turn);
          phase_barrier();
          fetch(j + 1 + turn);
          __builtin_amdgcn_s_setprio(1);
          values(j);
          scores(j + 1);  // (the last one's go nowhere)
          __builtin_amdgcn_s_setprio(0);
        }
      } else {
        for (int j = 0; j < tiles; ++j) {
          phase_barrier();
          stage(j + turn);
          phase_barrier();
          fetch(j + 1 + turn);
        }
      }
      if (!turn) phase_barrier();
    }

    // (worked out again: kept across the pages it costs registers that there are not)
    const int l2 = (int)opaque(threadIdx.x) & 63, lh2 = l2 >> 5, r = rb * kManyRows + 32 * wave + (l2 & 31);
    const float l = pair_sum(l_run);
    if (!PRE && !a.n_groups && i1 - i0 == n) {  // the rows' only piece
      const Row x = row_of<PRE>(a, seg, h, min(r, R - 1), si.hi);
      if (r < R && x.hi > 0) {
        store_rows(a.out + x.q_row * a.o_ld + (int64_t)x.head * kKv8Hd, o, l == 0.f ? 0.f : 1.0f / l, lh2);
        if (lh2 == 0) write_lse(a, x, m_run, l);
      }
    } else if (r < R) {
      const int64_t column = ((int64_t)h * n_seg + seg) * all_rb + rb;
      const int64_t slot = slot_of<PRE>(a, block, column, i0 == 0) * kManyRows + 32 * wave + (l2 & 31);
      if (lh2 == 0) {
        a.part[PRE].m[2 * slot] = m_run;
        a.part[PRE].m[2 * slot + 1] = l;
      }
      float* po = a.part[PRE].o + slot * kKv8Hd + 4 * lh2;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(po + 32 * db + 8 * i) =
              f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
    }
  }
}

// How a part's rows are worked on.
enum Kind { kNone, kFew16, kFew32, kMany };

// Wavefronts of a workgroup.
constexpr int waves_of(Kind prefix, Kind own) { return prefix == kMany || own == kMany ? kManyWaves : 4; }

// The own tokens' workgroups first: with a prefix of many rows theirs wait for memory
// while the others compute.
template <Kind PREFIX, Kind OWN>
__global__ void __launch_bounds__(waves_of(PREFIX, OWN) * 64, PREFIX <= kFew16 && OWN == kFew16 ? 3 : 2)
    kv8_pieces_kernel(const DecArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int W = waves_of(PREFIX, OWN);
  int* const few = reinterpret_cast<int*>(smem);
  const int block = blockIdx.x;
  if (PREFIX == kNone || block < a.part[0].blocks) {
    if constexpr (OWN == kMany) many_rows<false>(a, smem, block);
    if constexpr (OWN == kFew16) few_rows<W, 1, false>(a, few, block);
    if constexpr (OWN == kFew32) few_rows<W, 2, false>(a, few, block);
  } else {
    const int b = block - a.part[0].blocks;
    if constexpr (PREFIX == kMany) many_rows<true>(a, smem, b);
    if constexpr (PREFIX == kFew16) few_rows<W, 1, true>(a, few, b);
    if constexpr (PREFIX == kFew32) few_rows<W, 2, true>(a, few, b);
  }
}

// ------------------------------------------------------------------ join
// The pieces of a row: `n` of them, of the workers from w0 on.
struct Pieces {
  int n = 0, w0 = 0, rows = 0, r = 0;  // rows of a slot, and the row's place in it
  int64_t column = 0;
};
template <bool PRE>
__device__ __forceinline__ Pieces pieces_of(const DecArgs& a, int seg, int h, int r) {
  Pieces p;
  const Part& k = a.part[PRE];
  if (k.workers == 0) return p;
  const int n_seg = PRE ? a.n_groups : a.s.B, total = k.first[n_seg], from = k.first[seg], to = k.first[seg + 1];
  if (to == from) return p;
  const bool many = k.rows > kFewRows;
  int begin = h * total + from, n = to - from, rb = 0;
  if (many) {
    n /= row_blocks<PRE, true>(a, seg);
    rb = r / kManyRows;
    begin += rb * n;
  }
  const int run = many ? run_tiles<true>(total * a.Hkv, k.workers) : run_tiles<false>(total * a.Hkv, k.workers);
  p.w0 = begin / run;
  p.n = (begin + n - 1) / run - p.w0 + 1;
  p.rows = many ? kManyRows : k.rows;
  p.r = r - rb * kManyRows;
  p.column = ((int64_t)h * n_seg + seg) * (many ? (k.rows + kManyRows - 1) / kManyRows : 1) + rb;
  return p;
}
template <bool PRE>
__device__ __forceinline__ int64_t piece_row(const DecArgs& a, const Pieces& p, int x) {
  return slot_of<PRE>(a, p.w0 + x, p.column, x == 0) * p.rows + p.r;
}

// A row (b, t, query head) and its pieces; false where it was written as its only piece.
// (A call has less than 2^25 rows.)
struct JoinRow { Row w; Pieces own, pre; };
__device__ __forceinline__ bool find_row(const DecArgs& a, int row, JoinRow& j) {
  const int Hq = a.Hkv * a.G, tok = row / Hq, b = tok / a.s.T, t = tok - b * a.s.T;
  j.w.q_row = tok;
  j.w.head = row - tok * Hq;
  if (t >= kv8_len(a.s, b).fresh) return true;  // padding: no pieces, zeros and -inf
  const int h = j.w.head / a.G, r = t * a.G + j.w.head - h * a.G;
  j.own = pieces_of<false>(a, b, h, r);
  if (a.n_groups == 0) return j.own.n != 1;
  j.pre = pieces_of<true>(a, b / a.gs, h, (b % a.gs) * a.s.T * a.G + r);
  return true;
}

// The row by WAVES wavefronts: half a wavefront reads a piece's 128 values, weighed by
// their maxima.
template <int WAVES>
__device__ __forceinline__ void join_row(const DecArgs& a, int row) {
  __shared__ __attribute__((aligned(16))) float lds_o[4][kKv8Hd];
  __shared__ float lds_m[4], lds_l[4];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int share = wave % WAVES;  // of the row's wavefronts
  JoinRow j;
  if (!find_row(a, row, j)) return;
  const Row& w = j.w;
  const Pieces &own = j.own, &pre = j.pre;
  float M = kNoMax, L = 0.f;
  f32x4 acc{};
  const int all = pre.n + own.n;
  constexpr int kAhead = 4;
  for (int x0 = 2 * share + (lane >> 5); x0 < all; x0 += 2 * WAVES * kAhead) {
    float m[kAhead], l[kAhead];
    f32x4 o[kAhead];
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const int x = x0 + 2 * WAVES * y;
      m[y] = kNoMax;
      l[y] = 0.f;
      o[y] = f32x4{};
      if (x < all) {
        const bool p = x < pre.n;
        const int64_t at = p ? piece_row<true>(a, pre, x) : piece_row<false>(a, own, x - pre.n);
        const float* const ml = (p ? a.part[1].m : a.part[0].m) + 2 * at;
        m[y] = ml[0];
        l[y] = ml[1];
        o[y] = *reinterpret_cast<const f32x4*>((p ? a.part[1].o : a.part[0].o) + at * kKv8Hd + 4 * (lane & 31));
      }
    }
    float m_new = M;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) m_new = fmax_nc(m_new, m[y]);
    const float alpha = __builtin_amdgcn_exp2f(M - m_new);
    L *= alpha;
    acc *= alpha;
    M = m_new;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const float c = __builtin_amdgcn_exp2f(m[y] - M);
      L += l[y] * c;
      acc += o[y] * c;
    }
  }
  const float both = pair_max(M), c = __builtin_amdgcn_exp2f(M - both);
  M = both;
  L = pair_sum(L * c);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = pair_sum(acc[e] * c);
  if (WAVES > 1) {
    if (lane < 32) *reinterpret_cast<f32x4*>(&lds_o[wave][4 * lane]) = acc;
    if (lane == 0) {
      lds_m[wave] = M;
      lds_l[wave] = L;
    }
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int x = 1; x < WAVES; ++x) M = fmax_nc(M, lds_m[wave + x]);
    L = 0.f;
    acc = f32x4{};
#pragma unroll
    for (int x = 0; x < WAVES; ++x) {
      const float f = __builtin_amdgcn_exp2f(lds_m[wave + x] - M);
      L += lds_l[wave + x] * f;
      acc += *reinterpret_cast<const f32x4*>(&lds_o[wave + x][4 * (lane & 31)]) * f;
    }
  }
  if (lane < 32) write_row<4, 1>(a, w, &acc, M, L, lane);
}
// Many rows: eight by a wavefront. A lane each finds their pieces; half the wavefront
// then reads four rows' values, two pieces of each on their way: a row's lengths, pieces and
// values are loads that wait for each other.
template <bool PRE>
__global__ void __launch_bounds__(256) kv8_join_rows_kernel(const DecArgs a) {
  constexpr int kEach = 4, kAhead = 2;
  const int lane = threadIdx.x & 63, rows = a.s.B * a.s.T * a.Hkv * a.G;
  const int row0 = (blockIdx.x * 4 + uni(threadIdx.x >> 6)) * 2 * kEach, row = row0 + (lane & (2 * kEach - 1));
  JoinRow j{};
  bool mine = row < rows;
  if (mine) mine = find_row(a, row, j);
  const uint32_t todo = (uint32_t)__ballot(mine);
  if (!(todo & ((1 << 2 * kEach) - 1))) return;
  auto slot_rows = [&](int k) { return a.part[k].rows > kFewRows ? kManyRows : a.part[k].rows; };
  const int own_rows = slot_rows(0), pre_rows = PRE ? slot_rows(1) : 0;
  // pieces, of which the first n_pre are the prefix's; the first one's slot (less begins of slot_of)
  const int own_first = (int)slot_of<false>(a, j.own.w0, j.own.column, false);
  const int pre_first = PRE ? (int)slot_of<true>(a, j.pre.w0, j.pre.column, false) : 0;
  int n[kEach], n_pre[kEach], own_at[kEach], pre_at[kEach], own_r[kEach], pre_r[kEach], most = 0;
  float M[kEach], L[kEach];
  f32x4 acc[kEach];
#pragma unroll
  for (int y = 0; y < kEach; ++y) {
    const int from = 2 * y + (lane >> 5);
    n[y] = __shfl(j.own.n + j.pre.n, from);
    own_at[y] = __shfl(own_first, from);
    own_r[y] = __shfl(j.own.r, from);
    if (PRE) {
      n_pre[y] = __shfl(j.pre.n, from);
      pre_at[y] = __shfl(pre_first, from);
      pre_r[y] = __shfl(j.pre.r, from);
    }
    n[y] = (todo >> from) & 1 ? n[y] : 0;
    most = max(most, n[y]);
    M[y] = kNoMax;
    L[y] = 0.f;
    acc[y] = f32x4{};
  }
  for (int x0 = 0; __ballot(x0 < most); x0 += kAhead) {
    float m[kEach][kAhead], l[kEach][kAhead];
    f32x4 o[kEach][kAhead];
#pragma unroll
    for (int y = 0; y < kEach; ++y)
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        const int x = x0 + z;
        m[y][z] = kNoMax;
        l[y][z] = 0.f;
        o[y][z] = f32x4{};
        if (x < n[y]) {
          const bool p = PRE && x < n_pre[y];
          const int64_t at = p ? (int64_t)(pre_at[y] + x) * pre_rows + pre_r[y]
                           : PRE ? (int64_t)(own_at[y] + x - n_pre[y]) * own_rows + own_r[y]
                                 : (int64_t)(own_at[y] + 2 * x + (x == 0)) * own_rows + own_r[y];
          const float* const ml = (p ? a.part[1].m : a.part[0].m) + 2 * at;
          m[y][z] = ml[0];
          l[y][z] = ml[1];
          o[y][z] = *reinterpret_cast<const f32x4*>((p ? a.part[1].o : a.part[0].o) + at * kKv8Hd + 4 * (lane & 31));
        }
      }
#pragma unroll
    for (int y = 0; y < kEach; ++y) {
      const float m_new = fmax_nc(M[y], fmax_nc(m[y][0], m[y][1])), alpha = __builtin_amdgcn_exp2f(M[y] - m_new);
      L[y] *= alpha;
      acc[y] *= alpha;
      M[y] = m_new;
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        const float c = __builtin_amdgcn_exp2f(m[y][z] - m_new);
        L[y] += l[y][z] * c;
        acc[y] += o[y][z] * c;
      }
    }
  }
#pragma unroll
  for (int y = 0; y < kEach; ++y) {
    const int from = 2 * y + (lane >> 5);
    Row w{};
    w.q_row = __shfl((int)j.w.q_row, from);
    w.head = __shfl(j.w.head, from);
    if ((todo >> from) & 1) write_row<4, 1>(a, w, &acc[y], M[y], L[y], lane & 31);
  }
}

// A row by four wavefronts or one.
template <int WAVES>
__global__ void __launch_bounds__(256) kv8_join_kernel(const DecArgs a) {
  const int row = blockIdx.x * (4 / WAVES) + uni(threadIdx.x >> 6) / WAVES;
  if (row < a.s.B * a.s.T * a.Hkv * a.G) join_row<WAVES>(a, row);
}

// ------------------------------------------------------------------ host
// The work of a kind of segments: n_table pages at most, of which a window of `span`
// keys (0 = none) and the first `sinks` are seen. The chip is taken as it is (256 CUs), so
// that the workspace's size does not depend on the device that asks.
struct Deal {
  Kind kind = kNone;
  int64_t tiles = 0;  // at most
  int workers = 0, blocks = 0;
  int64_t slots = 0, slot_rows = 0, pages = 0;
};
Deal deal_of(int64_t n_table, int64_t span, int64_t sinks, int64_t rows, int64_t segments, int64_t heads, bool prefixes,
             bool beside_many) {
  Deal d;
  if (n_table == 0 || segments == 0 || rows == 0) return d;
  d.pages = span ? std::min(n_table, (span + kPage - 2) / kPage + 1 + cdiv(sinks, kPage)) : n_table;
  d.kind = rows <= 16 ? kFew16 : rows <= kFewRows ? kFew32 : kMany;
  const int64_t row_blocks = d.kind == kMany ? cdiv(rows, kManyRows) : 1, columns = segments * heads * row_blocks;
  d.tiles = columns * d.pages;
  if (d.kind == kMany) {
    d.blocks = d.workers = (int)std::min<int64_t>(cdiv(d.tiles, 2), 256);  // a workgroup a CU
    d.slot_rows = kManyRows;
  } else {
    const int waves = beside_many ? kManyWaves : 4;
    d.blocks = (int)std::min<int64_t>(cdiv(d.tiles, waves), 256 * (beside_many ? 1 : d.kind == kFew16 ? 3 : 2));
    d.workers = d.blocks * waves;
    d.slot_rows = rows;
  }
  d.slots = prefixes ? d.workers + columns : 2 * (int64_t)d.workers;
  return d;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// Both kinds of segments and the workspace's parts.
struct Plan {
  Deal d[2];
  int64_t rows[2];
  size_t o_at[2], m_at[2], first_at[2], bytes;
  int whole;  // wavefronts of kv8_whole_kernel, 0: pieces and their join
};
Plan plan(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d) {
  Plan p{};
  if (s->n_table == 0) return p;  // no tokens of their own, so no new ones: every row is padding
  const int64_t G = d->n_q_heads / c->n_kv_heads, S = d->sinks, H = c->n_kv_heads;
  const int64_t gs = d->n_groups ? s->B / d->n_groups : 0, segs[2] = {s->B, d->n_groups};
  p.rows[0] = (int64_t)s->T * G;
  p.rows[1] = gs * s->T * G;
  // keys that the rows of a segment see between them, at most
  p.d[1] = deal_of(d->n_prefix_table, d->window, S, p.rows[1], segs[1], H, true, false);
  p.d[0] = deal_of(s->n_table, d->window ? (int64_t)d->window + s->T - 1 : 0, S, p.rows[0], segs[0], H, d->n_groups > 0,
                   p.d[1].kind == kMany);
  if (d->n_groups == 0 && p.d[0].kind == kFew16 && p.d[0].pages <= (s->B * H >= 256 ? 32 : 24)) {
    p.whole = s->B * H <= 256 ? 8 : 4;
    return p;
  }
  for (int k = 0; k < 2; ++k) {
    if (p.d[k].kind == kNone) continue;
    const size_t rows = (size_t)p.d[k].slots * p.d[k].slot_rows;
    p.o_at[k] = p.bytes;
    p.bytes += round256(rows * kKv8Hd * 4);
    p.m_at[k] = p.bytes;
    p.bytes += round256(rows * 8);
    p.first_at[k] = p.bytes;
    p.bytes += round256((segs[k] + 1) * 4);
  }
  return p;
}

glt_status check_attn(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d, const char* who) {
  const glt_status r = check_kv8(c, s, who);
  if (r != GLT_OK) return r;
  GLT_CHECK(d, GLT_ERR_INVALID_ARG, "%s: null descriptor", who);
  GLT_CHECK(d->n_q_heads > 0 && d->n_q_heads % c->n_kv_heads == 0, GLT_ERR_SHAPE,
            "%s: n_q_heads=%d (a multiple of the cache's %d)", who, d->n_q_heads, c->n_kv_heads);
  GLT_CHECK(d->scale > 0.f && d->scale <= 3.4028234e38f, GLT_ERR_INVALID_ARG, "%s: scale %g must be positive and finite", who,
            (double)d->scale);
  GLT_CHECK(d->window >= 0 && d->sinks >= 0, GLT_ERR_INVALID_ARG, "%s: window=%d sinks=%d", who, d->window, d->sinks);
  GLT_CHECK(d->n_groups >= 0 && (d->n_groups == 0 || s->B % d->n_groups == 0), GLT_ERR_SHAPE,
            "%s: %d sequences in %d groups", who, s->B, d->n_groups);
  if (d->n_groups > 0) {
    GLT_CHECK(d->n_prefix_table >= 0 && d->n_prefix_table <= (1 << 23) && d->prefix_ld >= d->n_prefix_table, GLT_ERR_SHAPE,
              "%s: %d pages a prefix, rows %lld apart", who, d->n_prefix_table, (long long)d->prefix_ld);
    GLT_CHECK(d->prefix_lens && (d->prefix_pages || d->n_prefix_table == 0), GLT_ERR_INVALID_ARG, "%s: null pointer", who);
    GLT_CHECK(((uintptr_t)d->prefix_pages | (uintptr_t)d->prefix_lens) % 4 == 0, GLT_ERR_ALIGNMENT,
              "%s: tables and lengths must be 4-byte aligned", who);
  }
  // a launch holds less than 2^32 threads, 256 for a piece and head or 64 for a row
  const int64_t G = d->n_q_heads / c->n_kv_heads, rows = (int64_t)s->B * s->T * G;
  GLT_CHECK(rows < (1 << 25) / c->n_kv_heads, GLT_ERR_SHAPE, "%s: B=%d T=%d n_q_heads=%d", who, s->B, s->T, d->n_q_heads);
  if (s->B == 0 || s->T == 0) return GLT_OK;
  const Plan p = plan(c, s, d);
  for (int k = 0; k < 2; ++k)
    GLT_CHECK(p.d[k].tiles < INT32_MAX - (1 << 16), GLT_ERR_SHAPE, "%s: B=%d T=%d and tables of %d and %d pages", who, s->B,
              s->T, s->n_table, d->n_prefix_table);
  return GLT_OK;
}

typedef void (*Kernel)(DecArgs);
Kernel pieces_kernel(Kind prefix, Kind own) {
  // [prefix][own]: a prefix has at least its sequences' rows, and none where they have no tokens
  static const Kernel k[4][4] = {
      {nullptr, kv8_pieces_kernel<kNone, kFew16>, kv8_pieces_kernel<kNone, kFew32>, kv8_pieces_kernel<kNone, kMany>},
      {nullptr, kv8_pieces_kernel<kFew16, kFew16>, nullptr, nullptr},
      {nullptr, kv8_pieces_kernel<kFew32, kFew16>, kv8_pieces_kernel<kFew32, kFew32>, nullptr},
      {nullptr, kv8_pieces_kernel<kMany, kFew16>, kv8_pieces_kernel<kMany, kFew32>, kv8_pieces_kernel<kMany, kMany>}};
  return k[prefix][own];
}

// The dynamic-LDS limit is a per-device attribute of the kernels.
constexpr int kMaxSegLds = (8192 + 1) * 4;
glt_status set_limits(const char* who) {
  static std::atomic<bool> set[64];
  int dev = 0;
  GLT_TRY_HIP(hipGetDevice(&dev));
  GLT_CHECK(dev >= 0 && dev < 64, GLT_ERR_HIP, "%s: device index %d out of range", who, dev);
  if (set[dev].load(std::memory_order_acquire)) return GLT_OK;
  for (int p = kNone; p <= kMany; ++p)
    for (int o = kNone; o <= kMany; ++o)
      if (const Kernel f = pieces_kernel((Kind)p, (Kind)o); f && (p == kMany || o == kMany))
        GLT_TRY_HIP(hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, kManyLds + kMaxSegLds));
  GLT_TRY_HIP(hipFuncSetAttribute((const void*)kv8_whole_kernel<8>, hipFuncAttributeMaxDynamicSharedMemorySize, 8 * (128 + 16 * 512)));
  set[dev].store(true, std::memory_order_release);
  return GLT_OK;
}

glt_status launch(DecArgs& a, const Plan& p, const char* who, hipStream_t st) {
  const int64_t rows = (int64_t)a.s.B * a.s.T * a.Hkv * a.G;
  const glt_status r = set_limits(who);
  if (r != GLT_OK) return r;
  if (p.whole) {
    const size_t lds = p.whole * (128 + p.rows[0] * 512);
    const dim3 grid((unsigned)(a.s.B * a.Hkv));
    if (p.whole == 8) GLT_LAUNCH("kv8_whole", kv8_whole_kernel<8>, grid, dim3(512), lds, st, a);
    else GLT_LAUNCH("kv8_whole", kv8_whole_kernel<4>, grid, dim3(256), lds, st, a);
    GLT_LAUNCH_CHECK("kv8_whole");
    return GLT_OK;
  }
  if (const Kernel f = pieces_kernel(p.d[1].kind, p.d[0].kind)) {
    const int segs = std::max(p.d[0].kind ? a.s.B : 0, p.d[1].kind ? a.n_groups : 0);
    const size_t lds = (p.d[0].kind == kMany || p.d[1].kind == kMany ? kManyLds : 0) + (segs + 1) * 4;
    GLT_LAUNCH("kv8_pieces", f, dim3((unsigned)(p.d[0].blocks + p.d[1].blocks)), dim3(waves_of(p.d[1].kind, p.d[0].kind) * 64),
               lds, st, a);
    GLT_LAUNCH_CHECK("kv8_pieces");
  }
  // a wavefront a row against one for eight, us: 4160 rows 7.7, 10.6; 9600 9.5, 10.2; 16384
  // 12.5, 9.4; 32768 21.8, 13.1; 65536 43 (rows one after the other), 19, with nothing to
  // join 4.7 both; whole calls with prefixes, 15360 rows 70.5, 68, 102400 268, 219, 131072 460, 398
  if (rows <= 4096)
    GLT_LAUNCH("kv8_join", kv8_join_kernel<4>, dim3((unsigned)rows), dim3(256), 0, st, a);
  else if (rows <= 12288)
    GLT_LAUNCH("kv8_join", kv8_join_kernel<1>, dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, st, a);
  else if (a.n_groups)
    GLT_LAUNCH("kv8_join", kv8_join_rows_kernel<true>, dim3((unsigned)cdiv(rows, 32)), dim3(256), 0, st, a);
  else
    GLT_LAUNCH("kv8_join", kv8_join_rows_kernel<false>, dim3((unsigned)cdiv(rows, 32)), dim3(256), 0, st, a);
  GLT_LAUNCH_CHECK("kv8_join");
  return GLT_OK;
}

}  // namespace

}  // namespace glt

using namespace glt;

extern "C" size_t glt_kv8_attention_workspace_size(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d) {
  if (!c || !s || !d || s->B <= 0 || s->T <= 0 || c->n_kv_heads <= 0 || d->n_q_heads < c->n_kv_heads || s->n_table < 0 ||
      d->n_groups < 0 || d->window < 0 || d->sinks < 0 || (d->n_groups > 0 && d->n_prefix_table < 0))
    return 0;
  return plan(c, s, d).bytes;
}

extern "C" glt_status glt_kv8_attention(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d, const void* q,
                                        int64_t q_ld, void* out, int64_t o_ld, float* lse, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  static const char* who = "glt_kv8_attention";
  glt_status r = check_attn(c, s, d, who);
  if (r != GLT_OK || s->B == 0 || s->T == 0) return r;
  const int64_t lds[2] = {q_ld, o_ld};
  for (int i = 0; i < 2; ++i)
    GLT_CHECK(lds[i] >= (int64_t)d->n_q_heads * kKv8Hd && lds[i] % 8 == 0 && lds[i] < ((int64_t)1 << 31), GLT_ERR_SHAPE,
              "%s: %c_ld %lld (at least %d heads of %d, a multiple of 8)", who, "qo"[i], (long long)lds[i], d->n_q_heads, kKv8Hd);
  GLT_CHECK(q && out && lse, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(((uintptr_t)q | (uintptr_t)out) % 16 == 0 && (uintptr_t)lse % 4 == 0, GLT_ERR_ALIGNMENT,
            "%s: tensors must be 16-byte aligned", who);
  const Plan p = plan(c, s, d);
  const size_t need = p.bytes;
  GLT_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0), GLT_ERR_WORKSPACE,
            "%s: needs %zu workspace bytes, 256-byte aligned", who, need);
  const int64_t tokens = (int64_t)s->B * s->T, nq = 2 * kKv8Hd * (int64_t)d->n_q_heads;
  const ByteRows all[] = {{out, tokens, nq, 2 * o_ld},
                          dense_bytes(lse, tokens * d->n_q_heads * 4),
                          dense_bytes(workspace, (int64_t)need),
                          {q, tokens, nq, 2 * q_ld},
                          dense_bytes(c->data, (int64_t)glt_kv8_size(c->n_pages, c->n_kv_heads, c->head_dim))};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 5; ++j)
      GLT_CHECK(!overlap(all[i], all[j]), GLT_ERR_INVALID_ARG,
                "%s: out, lse and workspace must overlap neither each other nor q nor the cache", who);
  r = check_spared(s, all, 3, who);
  if (r != GLT_OK) return r;
  if (d->n_groups) {
    const ByteRows prefix[] = {table_bytes(d->prefix_pages, d->n_groups, d->prefix_ld, d->n_prefix_table),
                               dense_bytes(d->prefix_lens, 4 * (int64_t)d->n_groups)};
    for (int i = 0; i < 3; ++i)
      GLT_CHECK(!overlap(all[i], prefix[0]) && !overlap(all[i], prefix[1]), GLT_ERR_INVALID_ARG,
                "%s: results must overlap neither a prefix's pages nor its length", who);
  }

  DecArgs a{};
  a.cache = static_cast<const uint8_t*>(c->data);
  a.n_pages = c->n_pages;
  a.s = *s;
  a.n_groups = d->n_groups;
  a.gs = d->n_groups ? s->B / d->n_groups : 1;
  if (d->n_groups) {
    a.ppages = d->prefix_pages;
    a.plens = d->prefix_lens;
    a.prefix_ld = d->prefix_ld;
    a.n_prefix_table = d->n_prefix_table;
  }
  a.Hkv = c->n_kv_heads;
  a.G = d->n_q_heads / c->n_kv_heads;
  a.W = d->window;
  a.S = d->sinks;
  a.scale_log2 = d->scale * kLog2e;
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.q_ld = q_ld;
  a.o_ld = o_ld;
  for (int k = 0; k < 2; ++k) {
    char* const ws = static_cast<char*>(workspace);
    a.part[k] = {(int)p.rows[k], p.d[k].workers, p.d[k].blocks, reinterpret_cast<int*>(ws + p.first_at[k]),
                 reinterpret_cast<float*>(ws + p.o_at[k]), reinterpret_cast<float*>(ws + p.m_at[k])};
  }
  return launch(a, p, who, as_stream(stream));
}

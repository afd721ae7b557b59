// Attention of new tokens over the 8-bit cache of keys and values, for gfx950.
//
// A key j of a segment (a sequence's own tokens, or a prefix that a group of
// sequences shares) is seen by a row at position p if
//   j <= p  and  (no window  or  j > p - window  or  j < sinks).
// The codes are whole numbers of 7 bits and a sign: bf16 holds them exactly, so
//   s = (q . code_k) step_k scale,   o += (p step_v) . code_v
// need one rounding, of p step_v, and no value of k or v is formed.
//
// A segment's keys are cut into pieces; a piece's output, maximum and sum go into the
// workspace, and a last kernel joins each row's pieces in order. Few rows a segment
// (new tokens x query heads of a kv head: kv8_few_kernel) or many
// (kv8_many_kernel); how each is cut stands there.
#include <algorithm>
#include <atomic>

#include "attention_dev.hpp"
#include "kv8.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

constexpr float kSlack = 8.0f;      // running-max slack (log2 units)
constexpr float kNoMax = -3.0e38f;  // maximum of a row that has seen nothing

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
  // [0] the sequences' own tokens, [1] prefixes: rows of a segment and head, pages
  // of a piece (1: kv8_few_kernel cuts by itself), pieces that a segment has at most,
  // and the pieces' results by slot and row
  int rows[2], chunk[2], n_max[2];
  int workers[2];      // wavefronts of kv8_few_kernel, 0 where kv8_many_kernel runs
  int* first[2];       // its pages before each segment, and in all
  float* part_o[2];    // 128 each
  float* part_m[2];    // maximum (log2 units) and sum
};

__device__ __forceinline__ int prefix_len(const DecArgs& a, int b) {
  return a.n_groups ? min(max(a.plens[b / a.gs], 0), a.n_prefix_table * kPage) : 0;
}

// What the segment's rows see of it: its first `hi` keys, of which those from `lo`
// on and the first `sunk`; the pieces ns before the window's and the window's from c0.
struct Sight {
  int hi, ns, c0, n;
  __device__ __forceinline__ int chunk_at(int piece) const { return piece < ns ? piece : c0 + piece - ns; }
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
  const int keys = a.chunk[PRE] * kPage;
  Sight r;
  r.hi = hi;
  const int end = (hi + keys - 1) / keys;
  r.c0 = min(lo / keys, end);
  r.ns = min((sunk + keys - 1) / keys, r.c0);
  r.n = r.ns + end - r.c0;
  return r;
}

// A row's sight within a segment: key j is seen if j < hi and (j >= lo or j < sunk).
struct Row {
  int hi, lo, sunk;
  int64_t q_row;  // (b * T + t) and its head, for q and the outputs
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
__device__ __forceinline__ int64_t page_id(const DecArgs& a, int seg, int p) {
  return PRE ? a.ppages[seg * a.prefix_ld + p] : a.s.pages[seg * a.s.pages_ld + p];
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

// -------------------------------------------------------------- few rows
// Up to 16 NB rows a segment and head. The pages that the segments' rows see, of all
// heads, are one list, of which each wavefront takes an equal run whatever the
// lengths; where a run enters another segment or head, a piece ends. A wavefront loads a
// page's codes with 16-byte loads straight into the operands of
//   S^T[key][row] = K . Q^T,  O^T[channel][row] += V^T . P^T
// (16 x 16 x 32), with the softmax between: no LDS, no barrier, and every code is
// converted once.
//
// Lane l: row l & 15 of a block of 16, g = l >> 4. The keys of score block (beta, a) are
// numbered so that the accumulators are the second product's operand as they stand:
// element e of lane group g is key 16 g + 8 a + 4 beta + e of the page.
constexpr int kFewWaves = 4;

// Pages of a wavefront's run.
__device__ __forceinline__ int run_pages(int total, int workers) { return max((total + workers - 1) / workers, 1); }

template <int NB, bool PRE>
__global__ void __launch_bounds__(kFewWaves * 64, NB == 1 ? 3 : 2) kv8_few_kernel(const DecArgs a) {
  extern __shared__ int first[];  // pages before each segment, and in all
  __shared__ int wave_sum[kFewWaves];
  const int tid = threadIdx.x, lane = tid & 63, r15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_seg = PRE ? a.n_groups : a.s.B, R = a.rows[PRE];

  int total = 0;
  for (int s0 = 0; s0 < n_seg; s0 += kFewWaves * 64) {
    const int s = s0 + tid, n = s < n_seg ? sight<PRE>(a, s).n : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (lane == 63) wave_sum[wave] = x;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      if (w < wave) before += wave_sum[w];
      total += wave_sum[w];
    }
    if (s < n_seg) first[s] = before + x - n;
    __syncthreads();
  }
  total = __builtin_amdgcn_readfirstlane(total);
  if (blockIdx.x == 0) {  // for the join
    for (int s = tid; s < n_seg; s += kFewWaves * 64) a.first[PRE][s] = first[s];
    if (tid == 0) a.first[PRE][n_seg] = total;
  }

  const int worker = blockIdx.x * kFewWaves + wave, all = total * a.Hkv, run = run_pages(all, a.workers[PRE]);
  int at = worker * run;  // workers * run stays below all + workers
  const int stop = min(at + run, all);
  while (at < stop) {
    const int h = at / total, pos = at - h * total;
    int seg = 0;  // the last segment that starts at or before pos
    for (int end = n_seg; end - seg > 1;) {
      const int mid = (seg + end) >> 1;
      if (__builtin_amdgcn_readfirstlane(first[mid]) <= pos) seg = mid;
      else end = mid;
    }
    const Sight si = sight<PRE>(a, seg);
    const int i0 = pos - __builtin_amdgcn_readfirstlane(first[seg]), i1 = min(si.n, i0 + stop - at);  // of the segment's list
    at += i1 - i0;

    // (what depends on the lane is worked out for each run: kept, it costs registers
    // that there are not)
    const int l1 = (int)opaque(threadIdx.x) & 63;
    Row row[NB];
    bf16x8 qf[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = 16 * nb + (l1 & 15);
      row[nb] = row_of<PRE>(a, seg, h, min(r, R - 1), si.hi);
      const uint16_t* qp = a.q + row[nb].q_row * a.q_ld + (int64_t)row[nb].head * kKv8Hd + 16 * (l1 >> 4);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        qf[nb][s] = __builtin_bit_cast(bf16x8, row[nb].hi > 0 ? *reinterpret_cast<const u32x4*>(qp + 64 * (s >> 1) + 8 * (s & 1))
                                                              : u32x4{0u, 0u, 0u, 0u});
    }
    f32x4 o[NB][8];
    float m_run[NB], l_run[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m_run[nb] = kNoMax;
      l_run[nb] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[nb][i] = f32x4{};
    }

    int ids = 0;  // lane x: the id of the run's page i0 + x, 64 at a time
    for (int i = i0; i < i1; ++i) {
      const int x = (i - i0) & 63;
      if (x == 0) ids = i + lane < i1 ? (int)page_id<PRE>(a, seg, si.chunk_at(i + lane)) : 0;
      const int64_t id = __builtin_amdgcn_readlane(ids, x);
      const int p = si.chunk_at(i);
      const bool ok = id >= 0 && id < a.n_pages;
      const uint8_t* pg = a.cache + ((ok ? id : 0) * a.Hkv + h) * kHeadB;
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
      if (!ok)
#pragma unroll
        for (int i = 0; i < 2; ++i) kst[i] = vst[i] = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
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
        // the lanes' rows see the whole page (of others, lanes' columns are zeros)
        const bool whole = __all(p * kPage + kPage <= w.hi && (p * kPage >= w.lo || p * kPage + kPage <= w.sunk));
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nb][blk][e] *= step(kst, 8 * (blk & 1) + 4 * (blk >> 1) + e) * a.scale_log2;
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
        if (__any(mt > m_run[nb] + kSlack)) {
          const float m_new = fmax_nc(m_run[nb], mt);
          const float alpha = __builtin_amdgcn_exp2f(m_run[nb] - m_new);
          m_run[nb] = m_new;
          l_run[nb] *= alpha;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[nb][i] *= alpha;
        }
        float pv[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __builtin_amdgcn_exp2f(s[nb][i >> 2][i & 3] - m_run[nb]);
          l_run[nb] += x;
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

    const int l2 = (int)opaque(threadIdx.x) & 63, c15 = l2 & 15, cg = l2 >> 4;
    const int64_t slot = (int64_t)worker + (int64_t)h * n_seg + seg;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float l = quad_sum(l_run[nb]);
      const int r = 16 * nb + c15;
      if (r < R) {
        float* to = a.part_o[PRE] + (slot * R + r) * kKv8Hd + 4 * cg;
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<f32x4*>(to + 16 * i) = o[nb][i];
        if (cg == 0) {
          a.part_m[PRE][2 * (slot * R + r)] = m_run[nb];
          a.part_m[PRE][2 * (slot * R + r) + 1] = l;
        }
      }
    }
  }
}

// ------------------------------------------------------------- many rows
// One workgroup of four wavefronts per (segment, head, 128 rows, piece); a wavefront
// owns 32 rows as in attention for training (attention_train.hip). A page is the tile:
// the workgroup's threads load its codes into registers while the tile before is worked
// on, convert them and write them to LDS in the order in which the products' operands are
// read (1 KB of 64 lanes each, padded so that the writes spread over the banks).
constexpr int kManyWaves = 4;
constexpr int kManyRows = 32 * kManyWaves;
constexpr int kKFrag = 1040, kVFrag = 1056;           // bytes of an operand of 64 lanes
constexpr int kVTile = 16 * kKFrag;                   // after the 16 of k
constexpr int kSteps = kVTile + 16 * kVFrag;          // f32 steps of k (times scale) and v
constexpr int kManyBuf = kSteps + 2 * kPage * 4;      // 34,048 bytes
constexpr int kManyLds = 2 * kManyBuf;

template <bool PRE>
__global__ void __launch_bounds__(kManyWaves * 64, 2) kv8_many_kernel(const DecArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = a.rows[PRE], nrb = (R + kManyRows - 1) / kManyRows;
  int id = blockIdx.x;
  const int h = id % a.Hkv;
  id /= a.Hkv;
  const int rb = id % nrb;
  id /= nrb;
  const int piece = id % a.n_max[PRE], seg = id / a.n_max[PRE];
  const Sight si = sight<PRE>(a, seg);
  if (piece >= si.n) return;
  const int chunk = si.chunk_at(piece);

  const int r = rb * kManyRows + 32 * wave + lq;
  const Row w = row_of<PRE>(a, seg, h, min(r, R - 1), si.hi);
  const bool live = r < R && w.hi > 0;
  // pages that the workgroup's rows read of the piece: the last of their keys
  int last = live ? w.hi : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) last = max(last, __shfl_xor(last, o));
  int* const lasts = reinterpret_cast<int*>(smem);
  if (lane == 0) lasts[wave] = last;
  __syncthreads();
  last = max(max(lasts[0], lasts[1]), max(lasts[2], lasts[3]));
  __syncthreads();
  const int p0 = chunk * a.chunk[PRE], p1 = min(min(p0 + a.chunk[PRE], (si.hi + kPage - 1) / kPage), (last + kPage - 1) / kPage);

  bf16x8 qf[8];
  load_rows(qf, a.q + w.q_row * a.q_ld + (int64_t)w.head * kKv8Hd, live, lh);
  f32x16 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16{};
  float m_run = kNoMax, l_run = 0.f;

  lds_char* const lds = (lds_char*)smem;
  u32x4 kx[2], vx[2];
  uint32_t st = 0;
  auto fetch = [&](int p) {
    const int64_t pid = __builtin_amdgcn_readfirstlane((int)page_id<PRE>(a, seg, p));
    const bool ok = pid >= 0 && pid < a.n_pages;
    const uint8_t* pg = a.cache + ((ok ? pid : 0) * a.Hkv + h) * kHeadB;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kx[i] = *reinterpret_cast<const u32x4*>(pg + 16 * (tid + 256 * i));
      vx[i] = *reinterpret_cast<const u32x4*>(pg + kVOff + 16 * (tid + 256 * i));
    }
    if (tid < 2 * kPage) {
      st = *reinterpret_cast<const uint16_t*>(pg + kKStepOff + 2 * tid);
      if (!ok) st = 0x7fc0u;
    }
  };
  // 16 codes of token q >> 3, channels 16 (q & 7) .., or of channel q >> 2 and 16 tokens
  auto stage = [&](lds_char* to) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = tid + 256 * i;
      {
        const int key = q >> 3, s = q & 7;
        lds_char* x = to + ((key >> 5) * 8 + s) * kKFrag + (key & 31) * 16;
        *(lds_bf16x8*)x = codes8(kx[i][0], kx[i][1]);
        *(lds_bf16x8*)(x + 512) = codes8(kx[i][2], kx[i][3]);
      }
      {
        const int d = q >> 2, s2 = q & 3;
        lds_char* x = to + kVTile + ((d >> 5) * 4 + s2) * kVFrag + (d & 31) * 16;
        *(lds_bf16x8*)x = codes8(vx[i][0], vx[i][1]);
        *(lds_bf16x8*)(x + 512) = codes8(vx[i][2], vx[i][3]);
      }
    }
    if (tid < 2 * kPage) {
      const float f = __uint_as_float(st << 16);
      *(__attribute__((address_space(3))) float*)(to + kSteps + 4 * tid) = tid < kPage ? f * a.scale_log2 : f;
    }
  };

  auto step = [&](int p, const lds_char* rd) {
    const int key0 = p * kPage;
    f32x16 s[2] = {f32x16{}, f32x16{}};
    const lds_char* kr = rd + lane * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i & 1] = mfma(*(const lds_bf16x8*)(kr + ((i & 1) * 8 + (i >> 1)) * kKFrag), qf[i >> 1], s[i & 1]);
    const lds_char* sp = rd + kSteps + 16 * lh;  // steps of keys 32 kb + 8 i + 4 lh + e
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 f = *(const lds_f32x4*)(sp + 128 * kb + 32 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kb][4 * i + e] *= f[e];
      }
    const bool whole = __all(!live || (key0 + kPage <= w.hi && (key0 >= w.lo || key0 + kPage <= w.sunk)));
    if (!whole)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = key0 + 32 * kb + 8 * (e >> 2) + 4 * lh + (e & 3);
          const bool in = (j < w.hi) & ((j >= w.lo) | (j < w.sunk));
          s[kb][e] = in ? s[kb][e] : -INFINITY;
        }
    float m2[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      m2[kb] = s[kb][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) m2[kb] = fmax_nc(m2[kb], s[kb][e]);
    }
    const float mt = pair_max(fmax_nc(m2[0], m2[1]));
    if (__any(mt > m_run + kSlack)) {
      const float m_new = fmax_nc(m_run, mt);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= alpha;
    }
    u32x4 pw[4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 f = *(const lds_f32x4*)(sp + kPage * 4 + 128 * kb + 32 * i);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = __builtin_amdgcn_exp2f(s[kb][4 * i + e] - m_run);
          l_run += y;
          x[e] = y * f[e];
        }
        if (!whole)  // an unseen key's step may be anything
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = s[kb][4 * i + e] == -INFINITY ? 0.f : x[e];
        pw[2 * kb + (i >> 1)][2 * (i & 1)] = pack2_rne(x[0], x[1]);
        pw[2 * kb + (i >> 1)][2 * (i & 1) + 1] = pack2_rne(x[2], x[3]);
      }
    const lds_char* vr = rd + kVTile + lane * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      o[i & 3] = mfma(*(const lds_bf16x8*)(vr + ((i & 3) * 4 + (i >> 2)) * kVFrag), __builtin_bit_cast(bf16x8, pw[i >> 2]), o[i & 3]);
  };

  if (p0 < p1) {
    fetch(p0);
    stage(lds);
  }
  for (int p = p0; p < p1; ++p) {
    __syncthreads();  // tile p is whole, and every wavefront is done with tile p - 1
    lds_char *x = lds + ((p - p0) & 1) * kManyBuf, *y = lds + (~(p - p0) & 1) * kManyBuf;
    if (p + 1 < p1) fetch(p + 1);
    step(p, x);
    if (p + 1 < p1) stage(y);
  }

  const float l = pair_sum(l_run);
  if (r >= R) return;
  const int64_t slot = (((int64_t)seg * a.Hkv + h) * a.n_max[PRE] + piece) * R + r;
  if (lh == 0) {
    a.part_m[PRE][2 * slot] = m_run;
    a.part_m[PRE][2 * slot + 1] = l;
  }
  float* to = a.part_o[PRE] + slot * kKv8Hd + 4 * lh;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(to + 32 * db + 8 * i) = f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
}

// ------------------------------------------------------------------ join
// The pieces of a row: `n` of them, `step` rows of results apart.
struct Pieces { int64_t at; int n; int64_t step; };
template <bool PRE>
__device__ __forceinline__ Pieces pieces_of(const DecArgs& a, int seg, int h, int r) {
  Pieces p{0, 0, a.rows[PRE]};
  if (a.n_max[PRE] == 0) return p;
  if (a.workers[PRE]) {
    const int n_seg = PRE ? a.n_groups : a.s.B, total = a.first[PRE][n_seg];
    const int from = a.first[PRE][seg], to = a.first[PRE][seg + 1];
    if (to > from) {
      const int run = run_pages(total * a.Hkv, a.workers[PRE]);
      const int w0 = (h * total + from) / run, w1 = (h * total + to - 1) / run;
      p.n = w1 - w0 + 1;
      p.at = ((int64_t)w0 + (int64_t)h * n_seg + seg) * a.rows[PRE] + r;
    }
  } else {
    p.n = sight<PRE>(a, seg).n;
    p.at = ((int64_t)seg * a.Hkv + h) * a.n_max[PRE] * a.rows[PRE] + r;
  }
  return p;
}

// WAVES wavefronts a row (b, t, query head): its pieces, prefix first, weighed by their
// maxima. Half a wavefront reads a piece's 128 values.
template <int WAVES>
__global__ void __launch_bounds__(256) kv8_join_kernel(const DecArgs a) {
  __shared__ __attribute__((aligned(16))) float lds_o[4][kKv8Hd];
  __shared__ float lds_l[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  const int part = wave % WAVES;  // of the row's wavefronts
  const int Hq = a.Hkv * a.G;
  if (i >= (int64_t)a.s.B * a.s.T * Hq) return;
  const int64_t tok = i / Hq;
  const int hq = (int)(i % Hq), b = (int)(tok / a.s.T), t = (int)(tok % a.s.T), h = hq / a.G;
  const Kv8Len len = kv8_len(a.s, b);
  Pieces p[2] = {{0, 0, 0}, {0, 0, 0}};
  if (t < len.fresh) {
    const int r = t * a.G + hq % a.G;
    p[0] = pieces_of<false>(a, b, h, r);
    if (a.n_groups) p[1] = pieces_of<true>(a, b / a.gs, h, (b % a.gs) * a.s.T * a.G + r);
  }
  float M = kNoMax;
#pragma unroll
  for (int k = 1; k >= 0; --k)
    for (int x = lane; x < p[k].n; x += 64) M = fmax_nc(M, a.part_m[k][2 * (p[k].at + x * p[k].step)]);
  M = quad_max(M);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) M = fmax_nc(M, __shfl_xor(M, o));
  f32x4 acc{};
  float L = 0.f;
#pragma unroll
  for (int k = 1; k >= 0; --k) {
#pragma unroll 4
    for (int x = 2 * part + (lane >> 5); x < p[k].n; x += 2 * WAVES) {
      const int64_t at = p[k].at + x * p[k].step;
      const float wgt = __builtin_amdgcn_exp2f(a.part_m[k][2 * at] - M);
      L += a.part_m[k][2 * at + 1] * wgt;
      acc += *reinterpret_cast<const f32x4*>(a.part_o[k] + at * kKv8Hd + 4 * (lane & 31)) * wgt;
    }
  }
  L = pair_sum(L);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = pair_sum(acc[e]);
  if (WAVES > 1) {
    if (lane < 32) *reinterpret_cast<f32x4*>(&lds_o[wave][4 * lane]) = acc;
    if (lane == 0) lds_l[wave] = L;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      acc += *reinterpret_cast<const f32x4*>(&lds_o[wave + w][4 * (lane & 31)]);
      L += lds_l[wave + w];
    }
  }
  const float f = L == 0.f ? 0.f : 1.0f / L;  // nothing seen: zeros and -inf; NaN stays
  if (lane < 32)
    *reinterpret_cast<u32x2a*>(a.out + tok * a.o_ld + (int64_t)hq * kKv8Hd + 4 * lane) =
        u32x2a{pack2_rne(acc[0] * f, acc[1] * f), pack2_rne(acc[2] * f, acc[3] * f)};
  if (lane == 0)
    a.lse[((int64_t)b * Hq + hq) * a.s.T + t] =
        L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host
constexpr int kFewRows = 32;  // rows that kv8_few_kernel takes

// How a kind of segments is cut: n_table pages at most, of which a window of `span`
// keys (0 = none) and the first `sinks` are seen. The chip's size is taken as it is
// (256 CUs): the workspace's size must not depend on the device that asks.
struct Cut { int chunk, n_max, workers; int64_t slots; };
Cut cut(int64_t n_table, int64_t span, int64_t sinks, int64_t rows, int64_t segments, int64_t heads) {
  if (n_table == 0 || segments == 0 || rows == 0) return {1, 0, 0, 0};
  auto most = [&](int64_t c) {  // pieces of c pages
    const int64_t n = cdiv(n_table, c);
    return span ? std::min(n, (span + c * kPage - 2) / (c * kPage) + 1 + cdiv(sinks, c * kPage)) : n;
  };
  if (rows <= kFewRows) {
    const int64_t pages = segments * heads * most(1), per_cu = kFewWaves * (rows <= 16 ? 3 : 2);
    const int workers = (int)(cdiv(std::min<int64_t>(pages, 256 * per_cu), kFewWaves) * kFewWaves);
    return {1, (int)most(1), workers, workers + segments * heads};
  }
  const int64_t groups = segments * heads * cdiv(rows, kManyRows);
  const int64_t c = std::max<int64_t>(4, cdiv(most(1), std::max<int64_t>(1, cdiv(1024, groups))));
  return {(int)c, (int)most(c), 0, segments * heads * most(c)};
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// Sizes of both kinds of segments and the workspace's parts.
struct Plan {
  Cut c[2];
  int64_t rows[2];
  size_t o_at[2], m_at[2], first_at[2], bytes;
};
Plan plan(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d) {
  Plan p{};
  const int64_t G = d->n_q_heads / c->n_kv_heads, S = d->sinks, H = c->n_kv_heads;
  const int64_t gs = d->n_groups ? s->B / d->n_groups : 0, segs[2] = {s->B, d->n_groups};
  p.rows[0] = (int64_t)s->T * G;
  p.rows[1] = gs * s->T * G;
  // keys that the rows of a segment see between them, at most
  p.c[0] = cut(s->n_table, d->window ? (int64_t)d->window + s->T - 1 : 0, S, p.rows[0], segs[0], H);
  p.c[1] = cut(d->n_prefix_table, d->window, S, p.rows[1], segs[1], H);
  for (int k = 0; k < 2; ++k) {
    p.o_at[k] = p.bytes;
    p.bytes += round256((size_t)p.c[k].slots * p.rows[k] * kKv8Hd * 4);
    p.m_at[k] = p.bytes;
    p.bytes += round256((size_t)p.c[k].slots * p.rows[k] * 8);
    p.first_at[k] = p.bytes;
    p.bytes += p.c[k].workers ? round256((segs[k] + 1) * 4) : 0;
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
  for (int k = 0; k < 2; ++k) {
    const int64_t segs = k ? d->n_groups : s->B, groups = segs * c->n_kv_heads;
    GLT_CHECK(p.c[k].workers ? groups * p.c[k].n_max < INT32_MAX - (1 << 16)
                             : groups * cdiv(p.rows[k], kManyRows) * p.c[k].n_max < (1 << 24),
              GLT_ERR_SHAPE, "%s: B=%d T=%d and tables of %d and %d pages", who, s->B, s->T, s->n_table, d->n_prefix_table);
  }
  return GLT_OK;
}

template <int NB, bool PRE>
glt_status launch_few(const DecArgs& a, hipStream_t st) {
  const size_t lds = (size_t)(PRE ? a.n_groups : a.s.B) * 4;
  GLT_LAUNCH("kv8_few", (kv8_few_kernel<NB, PRE>), dim3(a.workers[PRE] / kFewWaves), dim3(kFewWaves * 64), lds, st, a);
  GLT_LAUNCH_CHECK("kv8_few");
  return GLT_OK;
}

template <bool PRE>
glt_status launch_part(const DecArgs& a, hipStream_t st) {
  if (a.n_max[PRE] == 0) return GLT_OK;
  if (a.workers[PRE]) return a.rows[PRE] <= 16 ? launch_few<1, PRE>(a, st) : launch_few<2, PRE>(a, st);
  const int64_t segs = PRE ? a.n_groups : a.s.B;
  const int64_t grid = segs * a.n_max[PRE] * cdiv(a.rows[PRE], kManyRows) * a.Hkv;
  GLT_LAUNCH("kv8_many", kv8_many_kernel<PRE>, dim3((unsigned)grid), dim3(kManyWaves * 64), kManyLds, st, a);
  GLT_LAUNCH_CHECK("kv8_many");
  return GLT_OK;
}

}  // namespace

}  // namespace glt

using namespace glt;

extern "C" size_t glt_kv8_attention_workspace_size(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d) {
  if (!c || !s || !d || s->B <= 0 || s->T <= 0 || c->n_kv_heads <= 0 || d->n_q_heads < c->n_kv_heads || s->n_table < 0 ||
      d->n_groups < 0 || d->window < 0 || d->sinks < 0 || (d->n_groups > 0 && d->n_prefix_table < 0))
    return 256;
  return std::max<size_t>(plan(c, s, d).bytes, 256);
}

extern "C" glt_status glt_kv8_attention(const glt_kv8_cache* c, const glt_kv8_seqs* s, const glt_kv8_attn* d, const void* q,
                                        int64_t q_ld, void* out, int64_t o_ld, float* lse, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  static const char* who = "glt_kv8_attention";
  const glt_status r = check_attn(c, s, d, who);
  if (r != GLT_OK || s->B == 0 || s->T == 0) return r;
  const int64_t lds[2] = {q_ld, o_ld};
  for (int i = 0; i < 2; ++i)
    GLT_CHECK(lds[i] >= (int64_t)d->n_q_heads * kKv8Hd && lds[i] % 8 == 0 && lds[i] < ((int64_t)1 << 31), GLT_ERR_SHAPE,
              "%s: %c_ld %lld (at least %d heads of %d, a multiple of 8)", who, "qo"[i], (long long)lds[i], d->n_q_heads, kKv8Hd);
  GLT_CHECK(q && out && lse, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(((uintptr_t)q | (uintptr_t)out) % 16 == 0 && (uintptr_t)lse % 4 == 0, GLT_ERR_ALIGNMENT,
            "%s: tensors must be 16-byte aligned", who);
  const Plan p = plan(c, s, d);
  const size_t need = std::max<size_t>(p.bytes, 256);
  GLT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, GLT_ERR_WORKSPACE,
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

  int dev = 0;
  GLT_TRY_HIP(hipGetDevice(&dev));
  GLT_CHECK(dev >= 0 && dev < 64, GLT_ERR_HIP, "%s: device index %d out of range", who, dev);
  // the dynamic-LDS limit is a per-device attribute of the kernels
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    for (const void* f : {(const void*)kv8_many_kernel<false>, (const void*)kv8_many_kernel<true>})
      GLT_TRY_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kManyLds));
    attr_set[dev].store(true, std::memory_order_release);
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
    a.chunk[k] = p.c[k].chunk;
    a.n_max[k] = p.c[k].n_max;
    a.workers[k] = p.c[k].workers;
    a.first[k] = reinterpret_cast<int*>(static_cast<char*>(workspace) + p.first_at[k]);
    a.rows[k] = (int)p.rows[k];
    a.part_o[k] = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_at[k]);
    a.part_m[k] = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.m_at[k]);
  }
  const hipStream_t st = as_stream(stream);
  glt_status e = launch_part<true>(a, st);
  if (e == GLT_OK) e = launch_part<false>(a, st);
  if (e != GLT_OK) return e;
  const int64_t rows = tokens * d->n_q_heads;
  if (rows <= 4096)  // few rows of many pieces, mostly
    GLT_LAUNCH("kv8_join", kv8_join_kernel<4>, dim3((unsigned)rows), dim3(256), 0, st, a);
  else
    GLT_LAUNCH("kv8_join", kv8_join_kernel<1>, dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, st, a);
  GLT_LAUNCH_CHECK("kv8_join");
  return GLT_OK;
}

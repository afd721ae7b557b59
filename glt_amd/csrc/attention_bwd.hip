// Attention backward for gfx950: the gradients of
//   s = scale q . k^T (masked), p = exp(s - lse), out = p . v
// with the probabilities recomputed from q, k and the forward's lse:
//   D  = rowsum(dout * out)           (= rowsum(p * dp))
//   dp = dout . v^T,  ds = p (dp - D)
//   dq = scale ds . k,  dk = scale ds^T . q,  dv = p^T . dout
// (k and v gradients summed over the query heads of their group.)
//
// Two kernels, no atomics: attn_dq_kernel owns query rows and walks the keys
// (three products), attn_dkdv_kernel owns key rows and walks the queries of
// every head of the group (four products). Seven products instead of the five
// of one pass, but every sum has one fixed order: a pass that owns key rows
// would add dq from many workgroups at once.
//
// In both, a wavefront owns 32 rows whose operands (q and dout, or k and v) and
// accumulators stay in registers; the rows that it walks come through LDS in
// tiles of 64, loaded once (direct to LDS, double buffered) and read in both
// directions that the products need (attention_dev.hpp). The score products
// are formed so that a lane holds one OWNED row: the packed p or ds is then the
// next product's operand as it stands in the accumulator's layout.
//
// p and ds are rounded to bf16, as the matrix instructions take them, all sums are
// f32: the gradients are off by 2.4 * 10^-3 in the 2-norm, of which their own
// rounding is 1.6.
//
// Long rows: matrix instructions run 0.52 (dq) and 0.59 (dkdv) of the time, at the
// power limit's 1.8 GHz. The rows in registers leave room for two wavefronts per
// SIMD, and a wavefront's own products depend on its
// exponentials, so one wavefront's arithmetic has to run beside the other's
// products. The two come from two workgroups of four, which nothing keeps in
// step. With one workgroup of eight instead (half the loads into LDS) they wait
// at the same barrier, and short rows leave more of them idle; dq + dkdv in us,
// 32 query and 8 kv heads, eight against four:
//   1 x 512 causal 73, 55;  6 x 777 causal 213, 188;  1 x 1024 causal 99, 74;
//   4 x 2048 causal 515, 498;  2 x 4096 causal 864, 849;  full 1568, 1579.
// At 2 x 4096 causal dq and dkdv take 385 and 464 us at best, 1.07 and 1.18 * 10^15
// operations a second of the unmasked part (a large library product: 1.24 *
// 10^15), and the whole backward 926 to 963 from machine to machine; 22 of dq's go
// into watching D's error (kOff). With few tokens the chip is not full (1 x 512
// launches 128 workgroups), and blocks of at most 512 keys are walked twice: the
// whole of 1 x 512 59 us, 1 x 1024 78, 4 x 2048 563.
#include <algorithm>
#include <atomic>

#include "attention_dev.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

// Key tiles up to which a block of rows takes D from its own probabilities.
constexpr int kExactTiles = 8;
// Error of a longer row's D, relative to the 2-norm of its ds, that is put right
// in dq: the roundings of p and out leave 2^-9 in flat rows. Without the second
// walk rows of one heavy key (T 700, scores of deviation 16) bring dq's error to
// 3.0 * 2^-9 and dk's to 2.9 * 2^-9, with it to 2.0 and 1.2.
constexpr float kOff = 0x1p-5f;

struct BwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* out;
  const uint16_t* dout;
  const float* lse;    // [B, Hq, T]
  float* stats;        // [2][B, Hq, T]: lse log2(e) and -D, written by the dq kernel
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float* part;         // Hq > Hkv: dk, dv by query head, [2][B, T, Hq, 128]
  const int32_t* seq_lens;
  int64_t q_ld, k_ld, v_ld, o_ld;
  int B, T, Hq, Hkv, causal;
  float scale;
};

// D of the lane's row: the diagonal of out . dout^T.
__device__ __forceinline__ float row_delta(const uint16_t* out_row, bool live, const bf16x8* dof, int lane) {
  const int lq = lane & 31, lh = lane >> 5;
  bf16x8 of[8];
  load_rows(of, out_row, live, lh);
  f32x16 x{};
#pragma unroll
  for (int s = 0; s < 8; ++s) x = mfma(of[s], dof[s], x);
  // row lq = 8 (lq >> 3) + 4 ((lq >> 2) & 1) + (lq & 3) of column lq
  const int e = 4 * (lq >> 3) + (lq & 3);
  float y = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) y = e == i ? x[i] : y;
  return pair_sum(((lq >> 2) & 1) == lh ? y : 0.f);
}

constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;  // rows that a workgroup owns

// Steps that fragments are read ahead of their matrix instructions: what the
// registers of each loop allow (dkdv holds two more sets of accumulators).
constexpr int kDqAhead = 4, kDkdvAhead = 2, kGradAhead = 2;

// ------------------------------------------------------------------- dq
// One workgroup per (batch, query head, block of 128 queries), longest rows
// first. LDS: two buffers of a K and a V tile (65 KB).
__global__ void __launch_bounds__(kWaves * 64, 2) attn_dq_kernel(const BwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, lq = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nqb = (a.T + kRows - 1) / kRows;
  const int rep = a.Hq / a.Hkv, nhb = a.Hq * a.B;
  const int id = blockIdx.x, hb = id % nhb;
  const int qb = nqb - 1 - id / nhb;
  const int g = hb % a.Hkv, h = g * rep + (hb / a.Hkv) % rep, b = hb / a.Hq;
  const int q0 = qb * kRows, wq0 = q0 + 32 * wave, myq = wq0 + lq;
  const int len = seq_len(a.seq_lens, b, a.T);
  const bool live = myq < len;
  const int kv_end = q0 >= len ? 0 : a.causal ? min(len, q0 + kRows) : len;
  const int ntiles = (kv_end + kTile - 1) / kTile;
  const int64_t tok = (int64_t)b * a.T + min(myq, a.T - 1);
  const int64_t stat = ((int64_t)b * a.Hq + h) * a.T + min(myq, a.T - 1);

  const __amdgpu_buffer_rsrc_t rk = uni_rsrc_a(a.k + (int64_t)b * a.T * a.k_ld + (int64_t)g * kHd, rows_extent(len, a.k_ld));
  const __amdgpu_buffer_rsrc_t rv = uni_rsrc_a(a.v + (int64_t)b * a.T * a.v_ld + (int64_t)g * kHd, rows_extent(len, a.v_ld));
  const uint32_t kb_ld = (uint32_t)(a.k_ld * 2), vb_ld = (uint32_t)(a.v_ld * 2);  // bytes
  const uint32_t kof = tile_lane_off(wave, lane, kb_ld), vof = tile_lane_off(wave, lane, vb_ld);
  lds_char* const lds = (lds_char*)smem;
  auto load = [&](int t, lds_char* dst) {
    load_tile<kWaves>(rk, dst, wave, kof, kb_ld, (uint32_t)t * kTile * kb_ld);
    load_tile<kWaves>(rv, dst + kTileB, wave, vof, vb_ld, (uint32_t)t * kTile * vb_ld);
  };
  if (ntiles > 0) load(0, lds);

  bf16x8 qf[8], dof[8];
  load_rows(qf, a.q + tok * a.q_ld + (int64_t)h * kHd, live, lh);
  load_rows(dof, a.dout + tok * a.o_ld + (int64_t)h * kHd, live, lh);
  const float lse2 = live ? a.lse[stat] * kLog2e : 0.f;
  float D = row_delta(a.out + tok * a.o_ld + (int64_t)h * kHd, live, dof, lane);

  const uint32_t ro = row_frag_off(lane), co = col_frag_off(lane);
  const float scale_log2 = a.scale * kLog2e;

  // Score products of key block kb (32 keys) of tile t: p in s, dp.
  auto probs = [&](int t, int kb, const lds_char* row, f32x16& s, f32x16& dp) {
    const int key0 = t * kTile + 32 * kb;
    score_product<kDqAhead>(row, qf, s, [](int) {});
    if (key0 + 32 > len || (a.causal && key0 + 31 > wq0)) {
      const int lim = (a.causal ? min(len, myq + 1) : len) - (key0 + 4 * lh);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) < lim ? s[e] : -INFINITY;
    }
    // the exponentials beside the other product
    score_product<kDqAhead>(row + kTileB, dof, dp, [&](int i) {
#pragma unroll
      for (int e = 2 * i; e < 2 * i + 2; ++e)
        s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale_log2, -lse2));
    });
  };
  // Walks the tiles; step u of the workgroup uses buffer u & 1. block(t, kb,
  // row, col) gets each 32-key block that this wavefront's rows read.
  const int mine = a.causal ? min(ntiles, (wq0 + 31) / kTile + 1) : ntiles;
  auto walk = [&](int u0, bool last, auto block) {
    auto next = [&](int t, lds_char* wr) {
      if (t + 1 < ntiles) load(t + 1, wr);
      else if (!last) load(0, wr);
    };
    auto step = [&](int t, const lds_char* __restrict__ rd, lds_char* __restrict__ wr) {  // K and V tile in rd
      next(t, wr);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int key0 = t * kTile + 32 * kb;
        if (key0 >= kv_end || (a.causal && key0 > wq0 + 31)) continue;
        block(t, kb, rd + opaque(ro + kb * 8 * kGroupB), rd + opaque(co + kb * 8 * kGroupB));
      }
    };
    for (int t = 0; t < ntiles; ++t) {
      __builtin_amdgcn_s_waitcnt(vmcnt_enc(0));
      phase_barrier();  // this step's tiles are whole, and every wavefront is done with the step before
      const int u = u0 + t;
      lds_char *x = lds + (u & 1) * 2 * kTileB, *y = lds + (~u & 1) * 2 * kTileB;
      if (t < mine) step(t, x, y);
      else next(t, y);
    }
  };

  // D from out carries out's rounding, which counts where few keys share a
  // row's weight: dp - D nearly cancels there. Blocks of few keys take it from
  // the probabilities, as D + sum p (dp - D), in a walk of their own.
  const bool exact = ntiles <= kExactTiles;
  int u = 0;
  if (exact) {
    float d = 0.f;
    walk(0, false, [&](int t, int kb, const lds_char* row, const lds_char*) {
      f32x16 s{}, dp{};
      probs(t, kb, row, s, dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) d = __builtin_fmaf(s[e], dp[e] - D, d);
    });
    D += pair_sum(d);
    u = ntiles;
  }

  f32x16 dq[4];
  float D_sum = 0.f;
  for (;;) {
    float sums = 0.f, squares = 0.f;  // of the row's ds
    f32x16 nD;  // where dp starts (16 subtractions less in each block)
#pragma unroll
    for (int e = 0; e < 16; ++e) nD[e] = -D;
    asm volatile("" : "+v"(nD));
#pragma unroll
    for (int i = 0; i < 4; ++i) dq[i] = f32x16{};
    walk(u, true, [&](int t, int kb, const lds_char* row, const lds_char* col) {
      f32x16 s{}, dp = nD;
      probs(t, kb, row, s, dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] *= dp[e];
        sums += s[e];
        squares = __builtin_fmaf(s[e], s[e], squares);
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const bf16x8 f = pack_frag(s, s2);
#pragma unroll
        for (int db = 0; db < 4; ++db) dq[db] = mfma(col_frag(col, db, s2), f, dq[db]);
      }
    });
    if (exact) {
      D_sum = D;
      break;
    }
    // With more keys the row's ds tell: their sum is what D is off by (dkdv gets
    // it without). Where that is more than kOff of their 2-norm the workgroup
    // walks once more with this row's D put right: rows of which one key has
    // some 0.95 of the weight (of flat ones it is 2^-9).
    if (u > 0) break;
    const float sum = pair_sum(sums);
    const bool off = live && sum * sum > kOff * kOff * pair_sum(squares);
    D_sum = D + sum;
    uint32_t* any = reinterpret_cast<uint32_t*>(smem + 4 * kTileB);
    const uint64_t offs = __ballot(off);
    if (lane == 0) any[wave] = offs != 0;
    phase_barrier();
    static_assert(kWaves == 4, "one flag a wavefront");
    if (!(any[0] | any[1] | any[2] | any[3])) break;
    D = off ? D_sum : D;
    u = ntiles;
    load(0, lds + (u & 1) * 2 * kTileB);
  }
  if (lh == 0 && myq < a.T) {
    a.stats[stat] = lse2;
    a.stats[(int64_t)a.B * a.Hq * a.T + stat] = live ? -D_sum : 0.f;
  }
  if (myq < a.T) {
    if (!live)
#pragma unroll
      for (int i = 0; i < 4; ++i) dq[i] = f32x16{};
    // a row that reads one key has no gradient on its score: not the rounding
    // that the product's order leaves (NaN stays)
    const bool one = myq == 0 && (a.causal || len == 1);
    store_rows(a.dq + tok * a.q_ld + (int64_t)h * kHd, dq, one ? 0.f : a.scale, lh);
  }
}

// ---------------------------------------------------------------- dk, dv
// One workgroup per (batch, query head, block of 128 keys), the blocks with the
// most queries first. LDS: two buffers of a Q and a dout tile and their 64 lse
// (times log2 e) and -D values. Where query heads share a kv head, each writes its
// f32 part and attn_dkdv_sum_kernel adds the parts in head order: a workgroup
// that walked the group's heads one after the other would leave too few
// workgroups for the chip (2 x 4096 tokens, 8 kv heads: 512 of very different
// length), and a cut that depends on the batch would make the sums' order depend
// on it. The parts cost 49 of 898 us at 2 x 4096 (268 MB written and read).
constexpr int kDkdvBuf = 2 * kTileB + 2 * kTile * 4;

__global__ void __launch_bounds__(kWaves * 64, 2) attn_dkdv_kernel(const BwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, lq = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rep = a.Hq / a.Hkv, nhb = a.Hq * a.B;
  const int id = blockIdx.x, hb = id % nhb, kb = id / nhb;
  const int g = hb % a.Hkv, h = g * rep + (hb / a.Hkv) % rep, b = hb / a.Hq;
  const int k0 = kb * kRows, wk0 = k0 + 32 * wave;
  const int len = seq_len(a.seq_lens, b, a.T);

  bf16x8 kf[8], vf[8];
  {
    const int64_t tok = (int64_t)b * a.T + min(wk0 + lq, a.T - 1);
    load_rows(kf, a.k + tok * a.k_ld + (int64_t)g * kHd, wk0 + lq < len, lane >> 5);
    load_rows(vf, a.v + tok * a.v_ld + (int64_t)g * kHd, wk0 + lq < len, lane >> 5);
  }

  // query tiles of this workgroup
  const int qt0 = a.causal ? k0 / kTile : 0;
  const int qt1 = k0 < len ? (len + kTile - 1) / kTile : qt0;
  const uint32_t qb_ld = (uint32_t)(a.q_ld * 2), ob_ld = (uint32_t)(a.o_ld * 2);  // bytes
  // rows at or past len read as zeros, lse and D too: p = 1 there, dp - D = 0
  // and dout = 0, so they add nothing
  const __amdgpu_buffer_rsrc_t rq = uni_rsrc_a(a.q + (int64_t)b * a.T * a.q_ld + (int64_t)h * kHd, rows_extent(len, a.q_ld));
  const __amdgpu_buffer_rsrc_t rdo = uni_rsrc_a(a.dout + (int64_t)b * a.T * a.o_ld + (int64_t)h * kHd, rows_extent(len, a.o_ld));
  const __amdgpu_buffer_rsrc_t rs = uni_rsrc_a(a.stats + ((wave & 1) * (int64_t)a.B * a.Hq + (int64_t)b * a.Hq + h) * a.T, (uint32_t)len * 4);
  lds_char* const lds = (lds_char*)smem;
  auto load = [&](int qt, lds_char* dst) {
    const int l = opaque(threadIdx.x) & 63;
    load_tile<kWaves>(rq, dst, wave, tile_lane_off(wave, l, qb_ld), qb_ld, (uint32_t)qt * kTile * qb_ld);
    load_tile<kWaves>(rdo, dst + kTileB, wave, tile_lane_off(wave, l, ob_ld), ob_ld, (uint32_t)qt * kTile * ob_ld);
    if (wave < 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(dst + 2 * kTileB + wave * kTile * 4), 4,
                                               (uint32_t)(qt * kTile + l) * 4, 0, 0, 0);
  };
  if (qt0 < qt1) load(qt0, lds);

  const uint32_t ro = row_frag_off(lane), co = col_frag_off(lane);
  f32x16 dk[4], dv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dk[i] = dv[i] = f32x16{};
  const float scale_log2 = a.scale * kLog2e;

  // tile qt, in rd (Q, dout, lse, D); tile qt + 1 into wr
  auto step = [&](int qt, const lds_char* __restrict__ rd, lds_char* __restrict__ wr) {
    if (qt + 1 < qt1) load(qt + 1, wr);
    const int q0t = qt * kTile;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const int q0 = q0t + 32 * qb;
      if (q0 >= len || (a.causal && q0 + 31 < wk0)) continue;
      f32x16 s{}, dp;
      const lds_char* row = rd + opaque(ro + qb * 8 * kGroupB);
      score_product<kDkdvAhead>(row, kf, s, [](int) {});
      if (a.causal && q0 < wk0 + 31) {  // row q0 + 8 (e >> 2) + 4 lh + (e & 3) reads keys up to itself
        const int l = opaque(threadIdx.x) & 63;
        const int lim = wk0 + (l & 31) - (q0 + 4 * (l >> 5));
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) >= lim ? s[e] : -INFINITY;
      }
      // the exponentials beside the other product; elements 4 i .. + 3 are
      // query rows 8 i + 4 lh .. + 3
      const lds_char* st = rd + opaque(2 * kTileB + 128 * qb + 16 * (lane >> 5));
      // the product starts at -D (16 subtractions less)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 D = *(const lds_f32x4*)(st + 32 * i + kTile * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * i + e] = D[e];
      }
      score_product<kDkdvAhead>(row + kTileB, vf, dp, [&](int i) {
        const f32x2 l = *(const lds_f32x2*)(st + 32 * (i >> 1) + 8 * (i & 1));
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s[2 * i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + e], scale_log2, -l[e]));
      });
      // a row that reads one key has no gradient on its score: not the rounding
      // that the product's order leaves (NaN stays)
      if (q0 == 0 && (a.causal || len == 1)) dp[0] = (opaque(threadIdx.x) & 32) || dp[0] != dp[0] ? dp[0] : 0.f;
      u32x4 pw[2], dw[2];  // packed p and ds
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int x = 4 * i + e, w = 2 * (i & 1) + e / 2;
          pw[i >> 1][w] = pack2_rne(s[x], s[x + 1]);
          dw[i >> 1][w] = pack2_rne(s[x] * dp[x], s[x + 1] * dp[x + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      const lds_char* col = rd + opaque(co + qb * 8 * kGroupB);
      __builtin_amdgcn_s_setprio(1);
      bf16x8 oa[kGradAhead], qa[kGradAhead];  // step i: 16 query rows i >> 2, d block i & 3
#pragma unroll
      for (int i = 0; i < kGradAhead; ++i) {
        oa[i] = col_frag(col + kTileB, i & 3, i >> 2);
        qa[i] = col_frag(col, i & 3, i >> 2);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dv[i & 3] = mfma(oa[i % kGradAhead], __builtin_bit_cast(bf16x8, pw[i >> 2]), dv[i & 3]);
        dk[i & 3] = mfma(qa[i % kGradAhead], __builtin_bit_cast(bf16x8, dw[i >> 2]), dk[i & 3]);
        if (i + kGradAhead < 8) {
          oa[i % kGradAhead] = col_frag(col + kTileB, (i + kGradAhead) & 3, (i + kGradAhead) >> 2);
          qa[i % kGradAhead] = col_frag(col, (i + kGradAhead) & 3, (i + kGradAhead) >> 2);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  };
  for (int qt = qt0; qt < qt1; ++qt) {
    __builtin_amdgcn_s_waitcnt(vmcnt_enc(0));
    phase_barrier();  // tile qt is whole, and every wavefront is done with tile qt - 1
    const int cur = (qt - qt0) & 1;
    step(qt, lds + cur * kDkdvBuf, lds + (cur ^ 1) * kDkdvBuf);
  }
  // the output rows' addresses are worked out again here: kept across the
  // loop they cost registers that it does not have
  const int tid = opaque(threadIdx.x);
  const int lh = (tid >> 5) & 1, myk = k0 + 32 * (tid >> 6) + (tid & 31);
  const int64_t tok = (int64_t)b * a.T + myk;
  if (myk >= a.T) return;
  if (myk >= len)
#pragma unroll
    for (int i = 0; i < 4; ++i) dk[i] = dv[i] = f32x16{};
  if (rep == 1) {
    store_rows(a.dk + tok * a.k_ld + (int64_t)g * kHd, dk, a.scale, lh);
    store_rows(a.dv + tok * a.v_ld + (int64_t)g * kHd, dv, 1.0f, lh);
    return;
  }
  float* pk = a.part + (tok * a.Hq + h) * kHd + 4 * lh;
  float* pv = pk + (int64_t)a.B * a.T * a.Hq * kHd;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f32x4*>(pk + 32 * db + 8 * i) = f32x4{dk[db][4 * i], dk[db][4 * i + 1], dk[db][4 * i + 2], dk[db][4 * i + 3]};
      *reinterpret_cast<f32x4*>(pv + 32 * db + 8 * i) = f32x4{dv[db][4 * i], dv[db][4 * i + 1], dv[db][4 * i + 2], dv[db][4 * i + 3]};
    }
}

// dk (blockIdx.y 0) or dv (1): the parts of a group's query heads added in head
// order, rounded once; a thread takes 8 elements of a token's kv head.
__global__ void __launch_bounds__(256) attn_dkdv_sum_kernel(const BwdArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int rep = a.Hq / a.Hkv, cols = a.Hkv * (kHd / 8);
  if (i >= (int64_t)a.B * a.T * cols) return;
  const int64_t row = i / cols;
  const int c = (int)(i - row * cols), g = c / (kHd / 8), e = c % (kHd / 8) * 8;
  const float* p = a.part + ((blockIdx.y ? (int64_t)a.B * a.T : 0) + row) * a.Hq * kHd + (int64_t)g * rep * kHd + e;
  f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
  for (int s = 1; s < rep; ++s) {
    x += *reinterpret_cast<const f32x4*>(p + s * kHd);
    y += *reinterpret_cast<const f32x4*>(p + s * kHd + 4);
  }
  const float f = blockIdx.y ? 1.0f : a.scale;
  uint16_t* dst = blockIdx.y ? a.dv + row * a.v_ld : a.dk + row * a.k_ld;
  *reinterpret_cast<u32x4*>(dst + g * kHd + e) =
      u32x4{pack2_rne(x[0] * f, x[1] * f), pack2_rne(x[2] * f, x[3] * f), pack2_rne(y[0] * f, y[1] * f),
            pack2_rne(y[2] * f, y[3] * f)};
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t stats_bytes(const glt_attn_desc* d) { return round256((size_t)2 * d->B * d->n_q_heads * d->T * sizeof(float)); }
size_t part_bytes(const glt_attn_desc* d) {
  return d->n_q_heads > d->n_kv_heads ? (size_t)2 * d->B * d->T * d->n_q_heads * kHd * sizeof(float) : 0;
}

glt_status launch_bwd(const BwdArgs& a, hipStream_t st) {
  constexpr int kDqLds = 4 * kTileB + 4 * kWaves, kDkdvLds = 2 * kDkdvBuf;
  // the dynamic-LDS limit is a per-device attribute of the kernels
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  GLT_TRY_HIP(hipGetDevice(&dev));
  GLT_CHECK(dev >= 0 && dev < 64, GLT_ERR_HIP, "glt_attention_bwd: device index %d out of range", dev);
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    GLT_TRY_HIP(hipFuncSetAttribute((const void*)attn_dq_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kDqLds));
    GLT_TRY_HIP(
        hipFuncSetAttribute((const void*)attn_dkdv_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kDkdvLds));
    attr_set[dev].store(true, std::memory_order_release);
  }
  const unsigned nb = (unsigned)cdiv(a.T, kRows);
  GLT_LAUNCH("attn_dq", attn_dq_kernel, dim3(nb * a.Hq * a.B), dim3(kWaves * 64), kDqLds, st, a);
  GLT_LAUNCH_CHECK("attn_dq");
  GLT_LAUNCH("attn_dkdv", attn_dkdv_kernel, dim3(nb * a.Hq * a.B), dim3(kWaves * 64), kDkdvLds, st, a);
  GLT_LAUNCH_CHECK("attn_dkdv");
  if (a.Hq > a.Hkv) {
    const int64_t chunks = (int64_t)a.B * a.T * a.Hkv * (kHd / 8);
    GLT_LAUNCH("attn_dkdv_sum", attn_dkdv_sum_kernel, dim3((unsigned)cdiv(chunks, 256), 2), dim3(256), 0, st, a);
    GLT_LAUNCH_CHECK("attn_dkdv_sum");
  }
  return GLT_OK;
}

}  // namespace

}  // namespace glt

using namespace glt;

extern "C" size_t glt_attention_bwd_workspace_size(const glt_attn_desc* d) {
  if (!d || d->B <= 0 || d->T <= 0 || d->n_q_heads <= 0 || d->n_kv_heads <= 0) return 256;
  return stats_bytes(d) + part_bytes(d);
}

extern "C" glt_status glt_attention_bwd(const glt_attn_desc* d, const void* q, const void* k, const void* v,
                                        const void* out, const float* lse, const void* dout, void* dq, void* dk,
                                        void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const glt_status s = check_attn_desc(d, "glt_attention_bwd");
  if (s != GLT_OK) return s;
  if (d->B == 0 || d->T == 0) return GLT_OK;
  GLT_CHECK(q && k && v && out && lse && dout && dq && dk && dv, GLT_ERR_INVALID_ARG, "glt_attention_bwd: null pointer");
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq |
                        (uintptr_t)dk | (uintptr_t)dv;
  GLT_CHECK(all % 16 == 0 && (uintptr_t)lse % 4 == 0 && (uintptr_t)d->seq_lens % 4 == 0, GLT_ERR_ALIGNMENT,
            "glt_attention_bwd: tensors must be 16-byte aligned");
  const size_t need = glt_attention_bwd_workspace_size(d);
  GLT_CHECK(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0, GLT_ERR_WORKSPACE,
            "glt_attention_bwd: needs %zu workspace bytes, 256-byte aligned", need);
  // every kernel reads inputs after others have written gradients
  const int64_t tokens = (int64_t)d->B * d->T, nq = 2 * kHd * d->n_q_heads, nk = 2 * kHd * d->n_kv_heads;
  const ByteRows in[] = {{q, tokens, nq, 2 * d->q_ld},   {k, tokens, nk, 2 * d->k_ld},    {v, tokens, nk, 2 * d->v_ld},
                         {out, tokens, nq, 2 * d->o_ld}, {dout, tokens, nq, 2 * d->o_ld}, dense_bytes(lse, tokens * d->n_q_heads * 4)};
  const ByteRows to[] = {{dq, tokens, nq, 2 * d->q_ld}, {dk, tokens, nk, 2 * d->k_ld}, {dv, tokens, nk, 2 * d->v_ld},
                         dense_bytes(workspace, (int64_t)need)};
  for (int i = 0; i < 4; ++i) {
    for (const ByteRows& x : in)
      GLT_CHECK(!overlap(to[i], x), GLT_ERR_INVALID_ARG, "glt_attention_bwd: gradients and workspace must overlap no input");
    for (int j = 0; j < i; ++j)
      GLT_CHECK(!overlap(to[i], to[j]), GLT_ERR_INVALID_ARG, "glt_attention_bwd: gradients and workspace must not overlap");
  }
  BwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<const uint16_t*>(out);
  a.dout = static_cast<const uint16_t*>(dout);
  a.lse = lse;
  a.stats = static_cast<float*>(workspace);
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(d));
  a.seq_lens = d->seq_lens;
  a.q_ld = d->q_ld; a.k_ld = d->k_ld; a.v_ld = d->v_ld; a.o_ld = d->o_ld;
  a.B = d->B; a.T = d->T; a.Hq = d->n_q_heads; a.Hkv = d->n_kv_heads;
  a.causal = d->causal; a.scale = d->scale;
  return launch_bwd(a, as_stream(stream));
}

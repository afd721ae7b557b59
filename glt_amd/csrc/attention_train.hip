// Causal GQA attention forward of a training step for gfx950: out and the
// log-sum-exp that the backward (attention_bwd.hip) recomputes the
// probabilities from. Row strides, sequence lengths of a padded batch.
//
// One workgroup of four wavefronts per (batch, query head, 128 query rows), the
// longest rows first; a wavefront owns 32 queries and walks tiles of 64 keys in
// LDS (attention_dev.hpp), a lane holding one query in every product:
//   S^T[key][q] = K . Q^T,  O^T[d][q] += V^T . P^T
// with the online softmax in between; K is read with its rows as the outer
// index, V with its rows contracted, in the order in which the accumulators of
// S^T hold them, so that the packed probabilities are the other operand as they
// stand. Two workgroups fit a CU, one wavefront of each per SIMD; as nothing
// keeps the two in step, one's arithmetic runs beside the other's products.
//
// The reads of a tile and the loads of the next go through distinct restrict
// pointers (step's rd and wr): without that the compiler lets every transposing
// read wait for all loads to LDS, the next tile's too (2 x 4096 causal 296 us).
//
// p is rounded to bf16, as the matrix instructions take it, the sums that divide
// and give lse are f32: out is off by 2.1 * 10^-3 in the 2-norm, of which its own
// rounding is 1.6.
//
// Long rows: matrix instructions run 0.54 of the time and vector ones 0.53, at the
// power limit's 1.8 GHz. 2 x 4096 causal with 32 query and 8 kv heads takes 260 to 277 us
// from machine to machine, 0.99 to 1.06 * 10^15 operations a second of the
// unmasked part, full 1.13 * 10^15 at best (a large library product: 1.24 * 10^15).
// Short ones: the longest rows' chain of tiles, 1.3 us each (1 x 512 15 us, 1 x
// 1024 24). us, against one workgroup of eight wavefronts (half the loads into
// LDS, but they wait at the same barrier):
//   1 x 512 causal 15, 19;  6 x 777 causal 55, 65;  1 x 1024 causal 24, 31;
//   4 x 2048 causal 148, 160;  2 x 4096 causal 260, 265;  2 x 4096 full 486, 484.
// Tiles of 32 keys let three wavefronts share a SIMD and measure the same within
// 5 % (6 x 777 52, 2 x 4096 full 497); longer read-ahead of the fragments
// changes nothing, without the raised priority of the second product 2 x 4096
// full takes 511.
#include <atomic>

#include "attention_dev.hpp"
#include "overlap.hpp"

namespace glt {

namespace {

constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;            // queries per workgroup
constexpr int kLds = 4 * kTileB;              // two buffers of a K and a V tile
constexpr float kSlack = 8.0f;                // running-max slack (log2 units)

struct FwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* lse;
  const int32_t* seq_lens;
  int64_t q_ld, k_ld, v_ld, o_ld;
  int B, T, Hq, Hkv, causal;
  float scale_log2;
  int window, sinks;  // WIN
};

// WIN: causal, and of the keys before it a row reads those less than `window`
// back and the first `sinks`. A block of 128 rows walks the sinks' tiles and those from
// its first row's window on: (window + 127) / 64 and one or two at the edges, whose masks cost
// 1 to 3 vector instructions a score. Blocks come in the sequence's order: they are of
// one length, but for the first ones, which so set the workgroups of a CU out of step
// (W 128: 59 us against 72). 2 x 4096, 32 query and 8 kv heads, window 1024 and 4
// sinks: 160 to 170 us, 0.71 to 0.75 * 10^15 operations a second of the visible part (0.88 of
// what the tiles hold); window 500 100 us, 128 56.
template <bool WIN>
__global__ void __launch_bounds__(kWaves * 64, 2) attn_train_fwd_kernel(const FwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, lq = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // query blocks longest first; (batch, head) with the kv head fastest, so that
  // an XCD's workgroups share kv heads
  const int nqb = (a.T + kRows - 1) / kRows;
  const int rep = a.Hq / a.Hkv, nhb = a.Hq * a.B;
  const int id = blockIdx.x, hb = id % nhb;
  const int qb = WIN ? id / nhb : nqb - 1 - id / nhb;
  const int g = hb % a.Hkv, h = g * rep + (hb / a.Hkv) % rep, b = hb / a.Hq;
  const int q0 = qb * kRows, wq0 = q0 + 32 * wave, myq = wq0 + lq;
  const int len = seq_len(a.seq_lens, b, a.T);
  const bool live = myq < len;
  const int kv_end = q0 >= len ? 0 : a.causal ? min(len, q0 + kRows) : len;
  const TileWalk<WIN> walk(q0, (kv_end + kTile - 1) / kTile, a.window, a.sinks);
  const int ntiles = walk.n;
  const int64_t tok = (int64_t)b * a.T + min(myq, a.T - 1);

  // keys at or past len read as zeros
  const __amdgpu_buffer_rsrc_t rk = uni_rsrc_a(a.k + (int64_t)b * a.T * a.k_ld + (int64_t)g * kHd, rows_extent(len, a.k_ld));
  const __amdgpu_buffer_rsrc_t rv = uni_rsrc_a(a.v + (int64_t)b * a.T * a.v_ld + (int64_t)g * kHd, rows_extent(len, a.v_ld));
  const uint32_t kb_ld = (uint32_t)(a.k_ld * 2), vb_ld = (uint32_t)(a.v_ld * 2);  // bytes
  const uint32_t kof = tile_lane_off(wave, lane, kb_ld), vof = tile_lane_off(wave, lane, vb_ld);
  lds_char* const lds = (lds_char*)smem;
  auto load = [&](int t, lds_char* dst) {
    const uint32_t row0 = (uint32_t)walk.tile(t) * kTile;
    load_tile<kWaves>(rk, dst, wave, kof, kb_ld, row0 * kb_ld);
    load_tile<kWaves>(rv, dst + kTileB, wave, vof, vb_ld, row0 * vb_ld);
  };
  if (ntiles > 0) load(0, lds);

  bf16x8 qf[8];
  load_rows(qf, a.q + tok * a.q_ld + (int64_t)h * kHd, live, lh);
  const uint32_t ro = row_frag_off(lane), co = col_frag_off(lane) + kTileB;

  f32x16 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16{};
  // running maximum (log2 units), sum of the rounded probabilities that the
  // output's product uses (its divisor), sum of the unrounded ones (lse's)
  float m_run = -3.0e38f, l_run = 0.f, l_exact = 0.f;

  // the walk's tile t, in rd (K, V); tile t + 1 into wr
  auto step = [&](int t, const lds_char* __restrict__ rd, lds_char* __restrict__ wr) {
    if (t + 1 < ntiles) load(t + 1, wr);
    const int key0 = walk.tile(t) * kTile;
    const lds_char *row = rd + opaque(ro), *col = rd + opaque(co);
    f32x16 s[2] = {f32x16{}, f32x16{}};  // key blocks 0, 1
    {
      constexpr int kAhead = 4;
      bf16x8 ka[kAhead];
      auto get = [&](int i) { return row_frag(row + (i & 1) * 8 * kGroupB, i >> 1); };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ka[i] = get(i);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i & 1] = mfma(ka[i % kAhead], qf[i >> 1], s[i & 1]);
        if (i + kAhead < 16) ka[i % kAhead] = get(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // Masked with -inf, which no scale lifts; a live row's first tile holds a
    // key that it may read, so its running maximum is finite from then on. (With
    // a window it may not: the maximum stays where it starts and the
    // probabilities are zeros.)
    if (WIN) {
      // an edge at a time: few tiles have two
      const int base = key0 + 4 * lh;
      if (key0 + kTile > len || key0 + kTile - 1 > wq0) {
        const int lim = min(len, myq + 1) - base;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = (32 * kb + 8 * (e >> 2) + (e & 3)) < lim ? s[kb][e] : -INFINITY;
      }
      if (key0 <= wq0 + 31 - a.window && key0 + kTile > a.sinks) {
        const int from = myq - a.window + 1 - base, sunk = a.sinks - base;
        if (key0 >= a.sinks) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] = (32 * kb + 8 * (e >> 2) + (e & 3)) >= from ? s[kb][e] : -INFINITY;
        } else {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int i = 32 * kb + 8 * (e >> 2) + (e & 3);
              s[kb][e] = (i >= from) | (i < sunk) ? s[kb][e] : -INFINITY;
            }
        }
      }
    } else if (key0 + kTile > len || (a.causal && key0 + kTile - 1 > wq0)) {
      const int lim = (a.causal ? min(len, myq + 1) : len) - (key0 + 4 * lh);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = (32 * kb + 8 * (e >> 2) + (e & 3)) < lim ? s[kb][e] : -INFINITY;
    }
    float m2[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      m2[kb] = s[kb][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) m2[kb] = fmax_nc(m2[kb], s[kb][e]);
    }
    const float mt = pair_max(fmax_nc(m2[0], m2[1])) * a.scale_log2;
    // the maximum moves only when some lane's grows by more than kSlack: the
    // probabilities stay below 2^kSlack, and the sums are rescaled on few tiles
    if (__any(mt > m_run + kSlack)) {
      const float m_new = fmax_nc(m_run, mt);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      l_exact *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= alpha;
    }
    u32x4 pw[4];  // packed probabilities of the four 16-key steps
    float ls[2] = {l_run, 0.f}, le[2] = {l_exact, 0.f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], a.scale_log2, -m_run));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e + 1], a.scale_log2, -m_run));
        const uint32_t w = pack2_rne(p0, p1);
        pw[2 * kb + (e >> 3)][(e & 7) >> 1] = w;
        ls[kb] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), kOnes2, ls[kb], false);
        le[kb] += p0 + p1;
      }
    l_run = ls[0] + ls[1];
    l_exact = le[0] + le[1];
    {
      constexpr int kAhead = 3;
      bf16x8 va[kAhead];
      auto get = [&](int i) { return col_frag(col, i & 3, i >> 2); };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) va[i] = get(i);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i & 3] = mfma(va[i % kAhead], __builtin_bit_cast(bf16x8, pw[i >> 2]), o[i & 3]);
        if (i + kAhead < 16) va[i % kAhead] = get(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  };
  const int mine = !WIN && a.causal ? min(ntiles, (wq0 + 31) / kTile + 1) : ntiles;  // tiles that this wavefront's rows read
  for (int t = 0; t < ntiles; ++t) {
    __builtin_amdgcn_s_waitcnt(vmcnt_enc(0));
    phase_barrier();  // tile t is whole, and every wavefront is done with tile t - 1
    lds_char *x = lds + (t & 1) * 2 * kTileB, *y = lds + (~t & 1) * 2 * kTileB;
    if (t < mine && walk.wanted(t, wq0, kTile)) step(t, x, y);
    else if (t + 1 < ntiles) load(t + 1, y);
  }

  const float l_tot = pair_sum(l_run), le = pair_sum(l_exact);
  if (myq >= a.T) return;
  // dead rows: zeros and -inf, whatever the lanes hold; a NaN sum gives NaN
  if (lh == 0)
    a.lse[((int64_t)b * a.Hq + h) * a.T + myq] =
        live ? (m_run + __builtin_amdgcn_logf(le)) * 0.6931471805599453f : -INFINITY;
  if (!live)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f32x16{};
  store_rows(a.out + tok * a.o_ld + (int64_t)h * kHd, o, !live || l_tot == 0.f ? 0.f : 1.0f / l_tot, lh);
}

}  // namespace

glt_status check_attn_desc(const glt_attn_desc* d, const char* who) {
  GLT_CHECK(d, GLT_ERR_INVALID_ARG, "%s: null descriptor", who);
  GLT_CHECK(d->B >= 0 && d->T >= 0 && d->n_q_heads > 0 && d->n_kv_heads > 0 && d->n_q_heads % d->n_kv_heads == 0,
            GLT_ERR_SHAPE, "%s: B=%d T=%d n_q_heads=%d n_kv_heads=%d (n_q_heads must be a multiple of n_kv_heads)", who,
            d->B, d->T, d->n_q_heads, d->n_kv_heads);
  GLT_CHECK(d->head_dim == kHd, GLT_ERR_UNSUPPORTED, "%s: head_dim %d (only %d)", who, d->head_dim, kHd);
  GLT_CHECK(d->scale > 0.f && d->scale <= 3.4028234e38f, GLT_ERR_INVALID_ARG, "%s: scale %g must be positive and finite",
            who, (double)d->scale);
  const int64_t lds[4] = {d->q_ld, d->k_ld, d->v_ld, d->o_ld};
  const int heads[4] = {d->n_q_heads, d->n_kv_heads, d->n_kv_heads, d->n_q_heads};
  for (int i = 0; i < 4; ++i) {
    GLT_CHECK(lds[i] >= (int64_t)heads[i] * kHd && lds[i] % 8 == 0, GLT_ERR_SHAPE,
              "%s: %c_ld %lld (at least %d heads of %d, a multiple of 8)", who, "qkvo"[i], (long long)lds[i], heads[i],
              kHd);
    // one sequence's rows, and the last tiles' past its end, are addressed
    // through 31-bit offsets
    GLT_CHECK(lds[i] < (int64_t)kOob && ((int64_t)d->T + 256) * lds[i] * 2 < (int64_t)kOob, GLT_ERR_SHAPE,
              "%s: T=%d rows of %c_ld %lld pass 2 GiB", who, d->T, "qkvo"[i], (long long)lds[i]);
  }
  // a launch holds less than 2^32 threads, 256 for 128 rows of a head or (the
  // sum of parts) 16 for a token's kv head
  GLT_CHECK(((int64_t)d->T + kRows - 1) / kRows * d->B < (1 << 24) / d->n_q_heads &&
                (int64_t)d->T * d->B < (1 << 28) / d->n_kv_heads,
            GLT_ERR_SHAPE, "%s: B=%d T=%d n_q_heads=%d n_kv_heads=%d", who, d->B, d->T, d->n_q_heads, d->n_kv_heads);
  return GLT_OK;
}

// Windows and sinks within a sequence of T; window 0 where it hides nothing.
glt_status check_window(const glt_attn_desc* d, int32_t* window, int32_t* sinks, const char* who) {
  GLT_CHECK(*window >= 1 && *sinks >= 0 && (*sinks <= kMaxSinks || *window >= d->T), GLT_ERR_INVALID_ARG,
            "%s: window %d (at least 1), sinks %d (0 to %d, or any with a window of T = %d or more)", who, *window, *sinks,
            kMaxSinks, d->T);
  GLT_CHECK(d->causal, GLT_ERR_UNSUPPORTED, "%s: a window is causal", who);
  if (*window >= d->T) *window = *sinks = 0;
  return GLT_OK;
}

namespace {

glt_status train_fwd(const glt_attn_desc* d, int32_t window, int32_t sinks, const void* q, const void* k, const void* v,
                     void* out, float* lse, void* stream, const char* who) {
  if (d->B == 0 || d->T == 0) return GLT_OK;
  GLT_CHECK(q && k && v && out && lse, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 == 0 && (uintptr_t)lse % 4 == 0 &&
                (uintptr_t)d->seq_lens % 4 == 0,
            GLT_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", who);
  // workgroups read keys and values that others' rows are written beside; a
  // query row is read by its own workgroup alone, before it writes
  const int64_t tokens = (int64_t)d->B * d->T, nq = 2 * kHd * d->n_q_heads, nk = 2 * kHd * d->n_kv_heads;
  const ByteRows rq{q, tokens, nq, 2 * d->q_ld}, rk{k, tokens, nk, 2 * d->k_ld}, rv{v, tokens, nk, 2 * d->v_ld},
      ro{out, tokens, nq, 2 * d->o_ld}, rl = dense_bytes(lse, tokens * d->n_q_heads * 4);
  GLT_CHECK(!overlap(ro, rk) && !overlap(ro, rv) && ((out == q && d->o_ld == d->q_ld) || !overlap(ro, rq)),
            GLT_ERR_INVALID_ARG, "%s: out must overlap no input (but q itself)", who);
  GLT_CHECK(!overlap(rl, rq) && !overlap(rl, rk) && !overlap(rl, rv) && !overlap(rl, ro), GLT_ERR_INVALID_ARG,
            "%s: lse must overlap no other tensor", who);
  // workgroups read lengths after others have written
  const ByteRows lens = dense_bytes(d->seq_lens, d->seq_lens ? 4 * (int64_t)d->B : 0);
  GLT_CHECK(!overlap(ro, lens) && !overlap(rl, lens), GLT_ERR_INVALID_ARG, "%s: out and lse must not overlap seq_lens", who);
  // the dynamic-LDS limit is a per-device attribute of the kernel
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  GLT_TRY_HIP(hipGetDevice(&dev));
  GLT_CHECK(dev >= 0 && dev < 64, GLT_ERR_HIP, "%s: device index %d out of range", who, dev);
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    for (const void* f : {(const void*)attn_train_fwd_kernel<false>, (const void*)attn_train_fwd_kernel<true>})
      GLT_TRY_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    attr_set[dev].store(true, std::memory_order_release);
  }
  FwdArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.seq_lens = d->seq_lens;
  a.q_ld = d->q_ld; a.k_ld = d->k_ld; a.v_ld = d->v_ld; a.o_ld = d->o_ld;
  a.B = d->B; a.T = d->T; a.Hq = d->n_q_heads; a.Hkv = d->n_kv_heads; a.causal = d->causal;
  a.scale_log2 = d->scale * kLog2e;
  a.window = window;
  a.sinks = sinks;
  const int64_t nblk = cdiv(d->T, kRows) * d->n_q_heads * d->B;
  if (window > 0)
    GLT_LAUNCH("attention_window", attn_train_fwd_kernel<true>, dim3((unsigned)nblk), dim3(kWaves * 64), kLds,
               as_stream(stream), a);
  else
    GLT_LAUNCH("attention_train", attn_train_fwd_kernel<false>, dim3((unsigned)nblk), dim3(kWaves * 64), kLds,
               as_stream(stream), a);
  GLT_LAUNCH_CHECK("attention_train");
  return GLT_OK;
}

}  // namespace

}  // namespace glt

using namespace glt;

extern "C" glt_status glt_attention_train_fwd(const glt_attn_desc* d, const void* q, const void* k, const void* v,
                                              void* out, float* lse, void* stream) {
  const glt_status s = check_attn_desc(d, "glt_attention_train_fwd");
  return s != GLT_OK ? s : train_fwd(d, 0, 0, q, k, v, out, lse, stream, "glt_attention_train_fwd");
}

extern "C" glt_status glt_attention_window_fwd(const glt_attn_desc* d, int32_t window, int32_t sinks, const void* q,
                                               const void* k, const void* v, void* out, float* lse, void* stream) {
  glt_status s = check_attn_desc(d, "glt_attention_window_fwd");
  if (s == GLT_OK) s = check_window(d, &window, &sinks, "glt_attention_window_fwd");
  return s != GLT_OK ? s : train_fwd(d, window, sinks, q, k, v, out, lse, stream, "glt_attention_window_fwd");
}

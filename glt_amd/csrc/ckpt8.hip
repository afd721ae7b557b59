// Activation checkpoints in 8 bits: what a training step saves for its
// backward, in 1 + 1/32 bytes a value instead of two (or four).
//
// A block is 32 consecutive columns of a row and shares one exponent byte E: the
// exponent field of the block's largest magnitude, one higher where that would
// round to more than 127 steps. A value is held as the byte 128 + rint(x /
// step), step = 2^(E - 133), so
//   * every step and every restored value is exact in f32 and bf16 (seven bits
//     and a power of two), the only rounding is to the nearest step (ties to
//     even): at most half a step, 1/127.5 of the block's largest magnitude
//     or, where that is more, 2^-134: steps end at 2^-133, E = 0;
//   * zero stays zero, and saving a restored block gives the same bytes (its
//     largest code is 64 or more, or E is 0, so its exponent is the same).
// E = 255: the block holds NaN or infinity and is restored as NaN. E = 254 is
// the last finite exponent; codes end at +-127 there. An integer code serves
// activations better than an 8-bit float of the same block: its error is
// uniform, a third of e4m3's over normal values (measured on N(0, 1): relative
// 2-norm 0.8 % against 2.9 %), and the block's exponent already carries the
// range.
//
// Layout of a checkpoint [rows, cols]: rows of codes, padded to whole blocks
// (code 128, zero), then from the next multiple of 256 bytes the exponents, row
// by row.
//
// All kernels stream and are bound by HBM: a thread takes a part of 8 columns, a
// quarter of a block, so that each of a wavefront's bf16 loads and stores covers
// whole lines (with 16 columns a thread each store wrote every other 16 bytes:
// gate, up and inter of 8192 x 15360 207 us against 155, which is 6.5 TB/s).
// 16384 x 4096 bf16: save 39 us, load 30 (5.2 and 6.8 TB/s, the codes partly from
// cache); 8192 x 4096 f32, whose stores are halves of lines that follow each other:
// save 24 us, load 27 (7.1 and 6.2 TB/s). Two or four parts a thread are no faster (save 39, 44), nor are
// non-temporal stores, which the reader of small activations would pay for.
#include "common.hpp"
#include "ckpt8.hpp"

namespace glt {

namespace {

constexpr int kThreads = 256;
constexpr int kVals = 8;   // values per thread

// 16 bytes at any element address (rows of an odd width start anywhere)
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Shape8 {
  uint32_t parts;   // of 8 columns per row, a multiple of four
  uint32_t total;   // of all rows
  int cols;
  int64_t ld;       // of the activation
  uint64_t exp_off; // bytes from the codes to the exponents
};

template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int cols, float* v) {
  constexpr int n = 16 / sizeof(T);
  if (c + kVals <= cols) {
#pragma unroll
    for (int q = 0; q < kVals / n; ++q) {
      const u32x4 x = *reinterpret_cast<const u32x4_any*>(row + c + q * n);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 2) {
          v[8 * q + 2 * w] = __uint_as_float(x[w] << 16);
          v[8 * q + 2 * w + 1] = __uint_as_float(x[w] & 0xFFFF0000u);
        } else {
          v[4 * q + w] = __uint_as_float(x[w]);
        }
      }
    }
    return;
  }
  // the row's end: the last element in the place of those past it, then zero
#pragma unroll
  for (int j = 0; j < kVals; ++j) {
    const T t = row[min(c + j, cols - 1)];
    float y;
    if constexpr (sizeof(T) == 2) y = bf16_to_f32(t);
    else y = t;
    v[j] = c + j < cols ? y : 0.f;
  }
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
}

template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const float* v) {
  if (c + kVals <= cols) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<u32x4_any*>(row + c) = u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        *reinterpret_cast<u32x4_any*>(row + c + 4 * q) =
            u32x4{__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                  __float_as_uint(v[4 * q + 3])};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVals; ++j)
    if (c + j < cols) {
      if constexpr (sizeof(T) == 2) row[c + j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
      else row[c + j] = v[j];
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) ckpt8_save_kernel(const T* __restrict__ x, uint8_t* __restrict__ ck, const Shape8 s) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= s.total) return;  // a block's four parts leave together
  const uint32_t row = i / s.parts, h = i - row * s.parts;
  float v[kVals];
  load8(x + (int64_t)row * s.ld, (int)h * kVals, s.cols, v);
  uint32_t top = 0;  // the largest magnitude's bits; NaN and infinity are larger than any number's
#pragma unroll
  for (int j = 0; j < kVals; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  // 127.5 steps and more carry into the exponent: mantissa 0x7F0000, below the
  // normal range, where no 1 stands before it, 0x7F8000
  const uint32_t E = top >= 0x7F800000u ? 255u : min((top + (top < 0x800000u ? 0x8000u : 0x10000u)) >> 23, 254u);
  uint32_t w[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(v[4 * q + j], 133 - (int)E), -127.f, 127.f);
      // rounded to an integer by the sum's own rounding, in its low bits
      b[j] = __float_as_uint(y + (12582912.f + 128.f));
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
    w[q] = E == 255u ? 0x80808080u : lo | hi;
  }
  *reinterpret_cast<u32x2*>(ck + (uint64_t)i * kVals) = u32x2{w[0], w[1]};
  if (!(h & 3)) ck[s.exp_off + (i >> 2)] = (uint8_t)E;
}

// The 8 values of part i.
__device__ __forceinline__ void restore8(const uint8_t* ck, const Shape8& s, uint32_t i, float* v) {
  const u32x2 w = *reinterpret_cast<const u32x2*>(ck + (uint64_t)i * kVals);
  const uint32_t E = ck[s.exp_off + (i >> 2)];
  const float step = E == 255u ? NAN : __builtin_amdgcn_ldexpf(1.0f, (int)E - 133);
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * q + j] = ((float)((w[q] >> (8 * j)) & 0xFFu) - 128.f) * step;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) ckpt8_load_kernel(const uint8_t* __restrict__ ck, T* __restrict__ x, const Shape8 s) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= s.total) return;
  const uint32_t row = i / s.parts, h = i - row * s.parts;
  float v[kVals];
  restore8(ck, s, i, v);
  store8(x + (int64_t)row * s.ld, (int)h * kVals, s.cols, v);
}

// gate, up and silu(gate) * up (in the order and with the sigmoid of the MLP's
// own epilogue) from the two checkpoints; inter for the columns of
// [lo, hi) only.
__global__ void __launch_bounds__(kThreads) ckpt8_swiglu_kernel(const uint8_t* __restrict__ g8, const uint8_t* __restrict__ u8,
                                                                uint16_t* __restrict__ gate, uint16_t* __restrict__ up,
                                                                uint16_t* __restrict__ inter, int lo, int hi, const Shape8 s) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= s.total) return;
  const uint32_t row = i / s.parts;
  const int c = (int)(i - row * s.parts) * kVals;
  const int64_t at = (int64_t)row * s.ld;
  float g[kVals], u[kVals];
  restore8(g8, s, i, g);
  restore8(u8, s, i, u);
  if (gate) store8(gate + at, c, s.cols, g);
  if (up) store8(up + at, c, s.cols, u);
  if (inter && c + kVals > lo && c < hi) {
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const float sg = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g[j] * 1.4426950408889634f));
      u[j] = g[j] * sg * u[j];
    }
    store8(inter + at, c, s.cols, u);
  }
}

uint64_t parts_of(int32_t cols) { return 4 * (uint64_t)(((int64_t)cols + 31) / 32); }
uint64_t code_bytes(int64_t rows, int32_t cols) { return (rows * parts_of(cols) * kVals + 255) / 256 * 256; }

glt_status check_shape(const char* who, int64_t rows, int32_t cols, int64_t ld, Shape8& s) {
  GLT_CHECK(rows >= 0 && cols > 0 && ld >= cols, GLT_ERR_SHAPE, "%s: rows=%lld cols=%d ld=%lld", who, (long long)rows, cols,
            (long long)ld);
  GLT_CHECK(rows < INT32_MAX && rows * (int64_t)parts_of(cols) < (1ll << 32) - kThreads, GLT_ERR_SHAPE,
            "%s: %lld rows of %d columns (at most 2^32 parts of 8)", who, (long long)rows, cols);
  s.parts = (uint32_t)parts_of(cols);
  s.total = (uint32_t)(rows * s.parts);
  s.cols = cols;
  s.ld = ld;
  s.exp_off = code_bytes(rows, cols);
  return GLT_OK;
}
dim3 grid8(const Shape8& s) { return dim3((s.total + kThreads - 1) / kThreads); }
bool off256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255) != 0; }
bool off_elem(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == GLT_DTYPE_F32 ? 4 : 2) != 0; }

}  // namespace

glt_status ckpt8_swiglu(const void* gate8, const void* up8, int64_t rows, int32_t cols, uint16_t* gate, uint16_t* up,
                        uint16_t* inter, int lo, int hi, hipStream_t st) {
  const char* who = "glt_ckpt8_swiglu";
  Shape8 s{};
  const glt_status e = check_shape(who, rows, cols, cols, s);
  if (e != GLT_OK) return e;
  if (rows == 0) return GLT_OK;
  GLT_CHECK(gate8 && up8, GLT_ERR_INVALID_ARG, "%s: null checkpoint", who);
  GLT_CHECK(!off256(gate8) && !off256(up8), GLT_ERR_ALIGNMENT, "%s: checkpoints must be 256-byte aligned", who);
  GLT_CHECK(!off_elem(gate, 0) && !off_elem(up, 0) && !off_elem(inter, 0), GLT_ERR_ALIGNMENT,
            "%s: pointers must be aligned to their elements", who);
  if (!gate && !up && !inter) return GLT_OK;
  GLT_LAUNCH("ckpt8_swiglu", ckpt8_swiglu_kernel, grid8(s), dim3(kThreads), 0, st, static_cast<const uint8_t*>(gate8),
             static_cast<const uint8_t*>(up8), gate, up, inter, lo, hi, s);
  GLT_LAUNCH_CHECK("ckpt8_swiglu");
  return GLT_OK;
}

}  // namespace glt

using namespace glt;

extern "C" {

size_t glt_ckpt8_size(int64_t rows, int32_t cols) {
  if (rows <= 0 || cols <= 0 || rows >= INT32_MAX) return 256;
  return code_bytes(rows, cols) + (rows * parts_of(cols) / 4 + 255) / 256 * 256;
}

glt_status glt_ckpt8_save(const void* x, int32_t dtype, int64_t ld, int64_t rows, int32_t cols, void* ckpt, void* stream) {
  const char* who = "glt_ckpt8_save";
  GLT_CHECK(dtype == GLT_DTYPE_BF16 || dtype == GLT_DTYPE_F32, GLT_ERR_DTYPE, "%s: dtype %d", who, dtype);
  Shape8 s{};
  const glt_status e = check_shape(who, rows, cols, ld, s);
  if (e != GLT_OK) return e;
  if (rows == 0) return GLT_OK;
  GLT_CHECK(x && ckpt, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(!off256(ckpt) && !off_elem(x, dtype), GLT_ERR_ALIGNMENT,
            "%s: the checkpoint must be 256-byte aligned, x to its element", who);
  uint8_t* ck = static_cast<uint8_t*>(ckpt);
  if (dtype == GLT_DTYPE_BF16)
    GLT_LAUNCH("ckpt8_save", ckpt8_save_kernel<uint16_t>, grid8(s), dim3(kThreads), 0, as_stream(stream),
               static_cast<const uint16_t*>(x), ck, s);
  else
    GLT_LAUNCH("ckpt8_save", ckpt8_save_kernel<float>, grid8(s), dim3(kThreads), 0, as_stream(stream),
               static_cast<const float*>(x), ck, s);
  GLT_LAUNCH_CHECK("ckpt8_save");
  return GLT_OK;
}

glt_status glt_ckpt8_load(const void* ckpt, int64_t rows, int32_t cols, void* x, int32_t dtype, int64_t ld, void* stream) {
  const char* who = "glt_ckpt8_load";
  GLT_CHECK(dtype == GLT_DTYPE_BF16 || dtype == GLT_DTYPE_F32, GLT_ERR_DTYPE, "%s: dtype %d", who, dtype);
  Shape8 s{};
  const glt_status e = check_shape(who, rows, cols, ld, s);
  if (e != GLT_OK) return e;
  if (rows == 0) return GLT_OK;
  GLT_CHECK(x && ckpt, GLT_ERR_INVALID_ARG, "%s: null pointer", who);
  GLT_CHECK(!off256(ckpt) && !off_elem(x, dtype), GLT_ERR_ALIGNMENT,
            "%s: the checkpoint must be 256-byte aligned, x to its element", who);
  const uint8_t* ck = static_cast<const uint8_t*>(ckpt);
  if (dtype == GLT_DTYPE_BF16)
    GLT_LAUNCH("ckpt8_load", ckpt8_load_kernel<uint16_t>, grid8(s), dim3(kThreads), 0, as_stream(stream), ck,
               static_cast<uint16_t*>(x), s);
  else
    GLT_LAUNCH("ckpt8_load", ckpt8_load_kernel<float>, grid8(s), dim3(kThreads), 0, as_stream(stream), ck,
               static_cast<float*>(x), s);
  GLT_LAUNCH_CHECK("ckpt8_load");
  return GLT_OK;
}

glt_status glt_ckpt8_swiglu(const void* gate8, const void* up8, int64_t rows, int32_t cols, uint16_t* gate, uint16_t* up,
                            uint16_t* inter, void* stream) {
  return ckpt8_swiglu(gate8, up8, rows, cols, gate, up, inter, 0, cols, as_stream(stream));
}

}  // extern "C"

// micro_common.cuh — what the microscaled kernels share: the formats, the quantisation of eight values per thread, the
// scale tiles' addresses, and vector access to fp16 / bf16 / fp32 rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdio>
#include <algorithm>
#include <exception>
#include <type_traits>
#include <utility>
#include <string>

#include "b2g.h"
#include "b2g_micro.h"

namespace b2g {

int32_t record_error(int32_t code, const std::string& msg);  // b2g_gemm.cu: sets b2g_last_error()

namespace micro {

enum Fmt : int { FMT_NONE = 0, FMT_MXFP8 = B2G_FMT_MXFP8, FMT_MXFP4 = B2G_FMT_MXFP4, FMT_NVFP4 = B2G_FMT_NVFP4 };

constexpr int block_of(int fmt) { return fmt == FMT_NVFP4 ? 16 : 32; }

// Nothing may be thrown across the C boundary: what a body throws (std::bad_alloc) becomes an error code.
template <typename F>
int32_t guarded(F&& body) {
  try {
    return body();
  } catch (const std::exception&) {
    return B2G_ERR_CUDA;
  }
}

inline int32_t launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return B2G_OK;
  return record_error(B2G_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int64_t min_pitch(int fmt, int64_t cols) { return ceil_div(cols, 32) * (fmt == FMT_MXFP8 ? 32 : 16); }

// Checks a microscaled tensor's fields; B2G_OK or an error with text naming `what`.
inline int32_t check_tensor(const b2g_micro_tensor* t, const char* what) {
  auto bad = [&](const char* why) { return record_error(B2G_ERR_INVALID_ARG, std::string(what) + ": " + why); };
  if (!t) return bad("null tensor");
  if (t->format < FMT_MXFP8 || t->format > FMT_NVFP4) return bad("format must be one of B2G_FMT_*");
  if (t->rows < 0 || t->cols < 0) return bad("negative dimension");
  if (t->rows >= (int64_t(1) << 31) - 128 || t->cols >= (int64_t(1) << 31) - 128)
    return record_error(B2G_ERR_UNSUPPORTED, std::string("dimension_too_large: ") + what + " needs rows and cols < 2^31 - 128");
  if (t->rows == 0 || t->cols == 0) return B2G_OK;
  if (!t->codes || !t->scales) return bad("null codes or scales");
  if (!aligned16(t->codes) || !aligned16(t->scales)) return bad("codes and scales must be 16-byte aligned");
  if (t->pitch < min_pitch(t->format, t->cols) || t->pitch % (t->format == FMT_MXFP8 ? 32 : 16))
    return bad("pitch too small or misaligned");
  if (t->format == FMT_NVFP4 && !t->scale) return bad("NVFP4 needs a tensor scale");
  return B2G_OK;
}

struct Mat {
  const void* p;
  int64_t sr, sc;
};

struct Quant {  // where a microscaled tensor goes
  uint8_t* codes;
  uint8_t* scales;
  const float* scale;
  int64_t pitch, ktiles, code_cols;
};

// How rows of `cols` values of `m` can be moved (Mode).
inline int mode_of(const b2g_micro_matrix* m, int64_t rows, int64_t cols, int64_t size) {
  if (m->stride_c != 1) return 2;
  return cols % 8 == 0 && aligned16(m->ptr) && (rows <= 1 || (m->stride_r * size) % 16 == 0) ? 0 : 1;
}

template <typename F>
int32_t by_mode(int mode, F&& f) {
  switch (mode) {
    case 0: return f(std::integral_constant<int, 0>{});
    case 1: return f(std::integral_constant<int, 1>{});
    default: return f(std::integral_constant<int, 2>{});
  }
}

inline Mat mat(const b2g_micro_matrix* m) { return Mat{m->ptr, m->stride_r, m->stride_c}; }

inline Quant quant(const b2g_micro_tensor* t) {
  return Quant{static_cast<uint8_t*>(t->codes), static_cast<uint8_t*>(t->scales), t->scale, t->pitch,
               ceil_div(t->cols, 4 * block_of(t->format)), ceil_div(t->cols, 32) * 32};
}

inline int32_t too_large(const char* what) {
  return record_error(B2G_ERR_UNSUPPORTED, std::string("dimension_too_large: ") + what + " needs fewer elements a call");
}

constexpr int64_t kMaxGrid = 2147483647;

// f(T{}, std::integral_constant<int, FMT>{}) for a value type and a format
template <typename F>
int32_t by_format(int fmt, F&& f) {
  switch (fmt) {
    case FMT_MXFP8: return f(std::integral_constant<int, FMT_MXFP8>{});
    case FMT_MXFP4: return f(std::integral_constant<int, FMT_MXFP4>{});
    default: return f(std::integral_constant<int, FMT_NVFP4>{});
  }
}

template <typename F>
int32_t by_flag(bool flag, F&& f) {
  return flag ? f(std::true_type{}) : f(std::false_type{});
}

template <typename F>
int32_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case B2G_VALUE_F16: return f(__half{});
    case B2G_VALUE_BF16: return f(__nv_bfloat16{});
    default: return f(float{});
  }
}

inline int32_t check_matrix(const b2g_micro_matrix* m, const char* what) {
  if (m && m->ptr) return B2G_OK;
  return record_error(B2G_ERR_INVALID_ARG, std::string("null ") + what);
}

// ---------------------------------------------------------------- device side
// Offset of the scale bytes of row `row` in tile column 0 of its row tile; tile column kt adds kt * 512.
__device__ __forceinline__ int64_t scale_row(int64_t row, int64_t ktiles) {
  return (row >> 7) * ktiles * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}

// Eight consecutive values of one row as they lie in memory: 16 bytes (fp16, bf16) or 32 (fp32).
template <typename T>
struct Raw8 {
  uint4 v;
};
template <>
struct Raw8<float> {
  uint4 v, w;
};

__device__ __forceinline__ float2 pair_f32(uint32_t w, __half*) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ float2 pair_f32(uint32_t w, __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&o)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_f32(w[i], static_cast<T*>(nullptr));
    o[2 * i] = f.x;
    o[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&o)[8]) {
  const uint32_t w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(w[i]);
}

__device__ __forceinline__ uint32_t pack_pair(float a, float b, __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float (&v)[8]) {
  T* t = nullptr;
  return Raw8<T>{make_uint4(pack_pair(v[0], v[1], t), pack_pair(v[2], v[3], t), pack_pair(v[4], v[5], t),
                            pack_pair(v[6], v[7], t))};
}
template <>
__device__ __forceinline__ Raw8<float> pack8<float>(const float (&v)[8]) {
  return Raw8<float>{make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])),
                     make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]))};
}

// How a row's values lie. kVec: unit column stride, 16-byte aligned rows and a multiple of 8 columns, so that eight
// columns exist or do not and are one or two 16-byte accesses. kUnit: unit column stride, any alignment and width: a
// warp moves 32 consecutive values an instruction and shared memory turns them to eight a lane (through strided
// scalars an odd width ran at a fifth of an even one's rate). kAny: any strides, a value at a time.
enum Mode : int { kVec = 0, kUnit = 1, kAny = 2 };

// A lane's eight columns c .. c+7 on their way from a row, columns at or past `cols` zero: `fetch` issues the loads,
// `settle` gives the values. In kUnit both are called by a converged warp whose lanes hold 256 consecutive columns,
// with a scratch of 256 values of the warp's own.
template <typename T, int MODE>
struct Frag {
  Raw8<T> r;
};
template <typename T>
struct Frag<T, kUnit> {
  T e[8];
};

template <typename T, int MODE>
__device__ __forceinline__ Frag<T, MODE> fetch8(const T* row, int64_t stride_c, int64_t c, int64_t cols) {
  Frag<T, MODE> f;
  if constexpr (MODE == kVec) {
    f.r.v = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (sizeof(T) == 4) f.r.w = f.r.v;
    if (c < cols) {
      const uint4* p = reinterpret_cast<const uint4*>(row + c);
      f.r.v = __ldg(p);
      if constexpr (sizeof(T) == 4) f.r.w = __ldg(p + 1);
    }
  } else if constexpr (MODE == kUnit) {
    const int lane = threadIdx.x & 31;
    const int64_t first = c - 7 * lane;  // c0 + lane of the warp's first column c0
#pragma unroll
    for (int i = 0; i < 8; ++i) f.e[i] = first + 32 * i < cols ? row[first + 32 * i] : from_f32<T>(0.f);
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32(row[(c + i) * stride_c]) : 0.f;
    f.r = pack8<T>(v);
  }
  return f;
}

template <typename T, int MODE>
__device__ __forceinline__ Raw8<T> settle8(const Frag<T, MODE>& f, T* scratch) {
  if constexpr (MODE == kUnit) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 8; ++i) scratch[32 * i + lane] = f.e[i];
    __syncwarp();
    const Raw8<T> r = reinterpret_cast<const Raw8<T>*>(scratch)[lane];
    __syncwarp();
    return r;
  } else {
    return f.r;
  }
}

template <typename T, int MODE>
__device__ __forceinline__ Raw8<T> load8(const T* row, int64_t stride_c, int64_t c, int64_t cols, T* scratch) {
  return settle8<T, MODE>(fetch8<T, MODE>(row, stride_c, c, cols), scratch);
}

template <typename T, int MODE>
__device__ __forceinline__ void store8(T* row, int64_t stride_c, int64_t c, int64_t cols, const Raw8<T>& r, T* scratch) {
  if constexpr (MODE == kVec) {
    if (c < cols) {
      uint4* p = reinterpret_cast<uint4*>(row + c);
      p[0] = r.v;
      if constexpr (sizeof(T) == 4) p[1] = r.w;
    }
  } else if constexpr (MODE == kUnit) {
    const int lane = threadIdx.x & 31;
    reinterpret_cast<Raw8<T>*>(scratch)[lane] = r;
    __syncwarp();
    const int64_t first = c - 7 * lane;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (first + 32 * i < cols) row[first + 32 * i] = scratch[32 * i + lane];
    __syncwarp();
  } else {
    float v[8];
    unpack8(r, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[(c + i) * stride_c] = from_f32<T>(v[i]);
  }
}

// The calling warp's scratch for kUnit (WARPS warps a block).
template <typename T, int MODE, int WARPS>
__device__ __forceinline__ T* warp_scratch() {
  if constexpr (MODE == kUnit) {
    __shared__ __align__(16) unsigned char scratch[WARPS * 256 * sizeof(T)];
    const int warp = (threadIdx.y * blockDim.x + threadIdx.x) >> 5;
    return reinterpret_cast<T*>(scratch) + warp * 256;
  } else {
    return nullptr;
  }
}

// The byte of a block's power-of-two scale: with amax = m * 2^e, the smallest exponent at which amax is at most the
// codes' largest magnitude (448 = 1.75 * 2^8, 6 = 1.5 * 2^2); from the bits alone, so it is exact. 255 (NaN) where the
// block holds an infinity or a NaN (their bits are above every finite magnitude's).
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  constexpr int emax = FMT == FMT_MXFP8 ? 8 : 2;
  constexpr uint32_t mant = FMT == FMT_MXFP8 ? 0x600000u : 0x400000u;
  const int e = static_cast<int>(amax_bits >> 23) - emax + ((amax_bits & 0x7fffffu) > mant ? 1 : 0);
  return amax_bits >= 0x7f800000u ? 255u : static_cast<uint32_t>(max(e, 0));
}

__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// A power-of-two scale's value (2^-127 is subnormal in fp32).
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
}

// Bits of the largest magnitude among eight values, as an fp32's; at least 0x7f800000 where an infinity or a NaN is
// among them. The integer pipe is what bounds the quantising kernels, so 16-bit values are compared as they lie, two
// at a time (magnitudes order as their bits do), and fp32 values by a maximum that takes the magnitude on the way,
// with a product by zero on the otherwise idle multiply-add pipe to catch what is not finite.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
__device__ __forceinline__ uint32_t max_magnitudes(const uint4& w) {  // of the even and the odd ones
  const uint32_t k = 0x7fff7fffu;
  return max_u16x2(max_u16x2(w.x & k, w.y & k), max_u16x2(w.z & k, w.w & k));
}
__device__ __forceinline__ uint32_t amax8(const Raw8<__nv_bfloat16>& r) {
  const uint32_t m = max_magnitudes(r.v);
  return max(m & 0xffff0000u, m << 16);
}
__device__ __forceinline__ uint32_t amax8(const Raw8<__half>& r) {
  const uint32_t m = max_magnitudes(r.v);
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m >> 16, m & 0xffffu)))));
}
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
  float m = 0.f, p = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, fabsf(v[i]));
    p = fmaf(v[i], 0.f, p);
  }
  return p == 0.f ? __float_as_uint(m) : 0x7fffffffu;
}
__device__ __forceinline__ uint32_t amax8(const Raw8<float>& r) {
  float v[8];
  unpack8(r, v);
  return amax8(v);
}

// One block's quantiser: its scale byte, and how an element becomes a code's value.
//   MX: x * 2^-e, exact unless it leaves fp32's range at the bottom, where the code is zero anyway.
//   NVFP4: x / u, u = block scale * tensor scale, correctly rounded as a division's quotient so that values on the
//   border between two codes fall as the definition says: one reciprocal a block, then per element the quotient's
//   estimate corrected by its residual (Markstein, "Computation of elementary functions on the IBM RISC System/6000
//   processor", 1990). The residual is taken negated, so that zeros keep the value's sign. A block whose scale rounds to
//   zero is zero.
// The codes of a NaN block are cleared by `keep`. NVFP4's tensor scale g as a thread uses it: 6 g and its reciprocal,
// once, so that a block's scale amax / (6 g) is three operations of the same kind. Residuals that would leave fp32's range
// at the bottom are avoided: below g = 2^-60 a block's scale is divided as such, and codes8 lifts values and u where u may
// be below 2^-100 (the last bit of a quotient above 2^-3, times that of u, is then below 2^-149).
struct TensorScale {
  float g, six, inv;
  __device__ __forceinline__ explicit TensorScale(float scale) : g(scale), six(6.f * scale), inv(1.f / (6.f * scale)) {}
  __device__ __forceinline__ float block(float amax) const {
    const float a = fminf(amax, 448.f * six);  // past it the scale saturates, and the quotient may leave fp32's range
    if (g < 8.67361738e-19f) return a / six;
    const float q = a * inv;
    return fmaf(-fmaf(q, six, -a), inv, q);
  }
};

template <int FMT>
struct BlockQuant {
  uint32_t byte;
  uint32_t keep;  // all ones; 0 in a NaN block
  float mul;      // MX: 2^-e; NVFP4: 1 / u, or 0
  float unit;     // NVFP4: u
  bool tiny;      // NVFP4: u may be below 2^-100, where a quotient's residual is among fp32's subnormals
  __device__ __forceinline__ void init(uint32_t amax_bits, const TensorScale& ts) {
    const bool bad = amax_bits >= 0x7f800000u;
    keep = bad ? 0u : 0xffffffffu;
    if constexpr (FMT == FMT_NVFP4) {
      byte = bad ? 0x7fu : __nv_cvt_float_to_fp8(ts.block(__uint_as_float(amax_bits)), __NV_SATFINITE, __NV_E4M3);
      unit = e4m3_to_f32(byte) * ts.g;
      tiny = ts.g < 4.03896783e-28f;  // 2^-91: block scales go down to 2^-9
      mul = byte == 0u ? 0.f : reciprocal(unit);
    } else {
      byte = mx_scale_byte<FMT>(amax_bits);
      mul = __uint_as_float((254u - byte) << 23);
    }
  }
  // 1 / u, the hardware's estimate corrected by its residual (Markstein, as above).
  __device__ __forceinline__ static float reciprocal(float u) {
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(u));
    return fmaf(-fmaf(u, y, -1.f), y, y);
  }
  __device__ __forceinline__ float scaled(float x) const {
    if constexpr (FMT == FMT_NVFP4) {
      const float q = x * mul;
      return fmaf(-fmaf(q, unit, -x), mul, q);
    } else {
      return x * mul;
    }
  }
};

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Eight e2m1 codes, the lowest value in the lowest bits: four conversions of two values to a byte and one packing
// move.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight values' codes: .x (and .y for MXFP8), lowest column in the lowest bits. EXACT: also with a tiny u, which only values
// that are quantised as they lie are worth (a layer's outputs carry errors of their own, and the norm takes 4 % longer).
template <int FMT, bool EXACT>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], BlockQuant<FMT> b) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = v[i];
  if constexpr (FMT == FMT_NVFP4) {
    // The largest scale: values past 6 u saturate, and their quotients may leave fp32's range. (No other scale's values
    // saturate.) A tiny u: the quotients are those of 2^40 times value and u, whose residuals fp32 holds.
    const bool tiny = EXACT && b.tiny;
    if (b.byte == 0x7eu || tiny) {
      const float top = b.byte == 0x7eu ? 8.f * b.unit : __uint_as_float(0x7f800000u);
      const float lift = tiny ? 1099511627776.f : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = fminf(fmaxf(s[i], -top), top) * lift;
      b.unit *= lift;
      b.mul *= 1.f / lift;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = b.scaled(s[i]);
  if constexpr (FMT == FMT_MXFP8)
    return make_uint2(e4m3x4(s[0], s[1], s[2], s[3]) & b.keep, e4m3x4(s[4], s[5], s[6], s[7]) & b.keep);
  else return make_uint2(e2m1x8(s) & b.keep, 0u);
}

// Where a lane's eight columns of a row go: eight consecutive columns per lane, the warp's 32 lanes holding 256 of one
// row (lane 0's first, a multiple of 256 past the row's start).
template <int FMT>
struct CodePlace {
  uint8_t* codes;   // the lane's codes in the row
  uint8_t* word;    // the scale word its block is in
  bool has_codes;   // the columns exist in the codes (below code_cols)
  bool leads;       // this lane stores the word, and the word exists
  __device__ __forceinline__ CodePlace(const Quant& q, int64_t row, int64_t c, int lane) {
    constexpr int kLanes = block_of(FMT) / 2;  // lanes that share a word: four blocks
    const int64_t kt = c / (4 * block_of(FMT));
    codes = q.codes + row * q.pitch + (FMT == FMT_MXFP8 ? c : c >> 1);
    word = q.scales + scale_row(row, q.ktiles) + kt * 512;
    has_codes = c < q.code_cols;
    leads = (lane & (kLanes - 1)) == 0 && kt < q.ktiles;
  }
};

// Quantise them. `m`: the eight values' amax8. A block's lanes (4 for blocks of 32, 2 for 16) share their largest
// magnitude by shuffles; the four scale bytes of one tile row are gathered into one 4-byte store. Called by a
// converged warp.
template <int FMT, bool EXACT>
__device__ __forceinline__ void quantize_store(const float (&v)[8], uint32_t m, int lane, const CodePlace<FMT>& to,
                                               const TensorScale& ts) {
  constexpr int kLanes = block_of(FMT) / 8;
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  BlockQuant<FMT> b;
  b.init(m, ts);
  const uint2 q = codes8<FMT, EXACT>(v, b);
  if (to.has_codes) {
    if constexpr (FMT == FMT_MXFP8) *reinterpret_cast<uint2*>(to.codes) = q;
    else *reinterpret_cast<uint32_t*>(to.codes) = q.x;
  }
  uint32_t w = b.byte << (8 * ((lane / kLanes) & 3));
  w |= __shfl_xor_sync(0xffffffffu, w, kLanes);
  w |= __shfl_xor_sync(0xffffffffu, w, 2 * kLanes);
  if (to.leads) *reinterpret_cast<uint32_t*>(to.word) = w;
}

}  // namespace micro
}  // namespace b2g

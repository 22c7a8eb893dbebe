// micro_quant.cu — quantisation into microscaled tensors and back, and the SiLU gate between two products.
//
// All of it moves bytes: the time is that of reading the values and writing codes and scales once. A warp's task is
// 256 columns of the four rows j, j + 32, j + 64, j + 96 of a 128-row scale tile: eight columns a lane, one 16-byte
// load a row, four loads in flight, and the four rows' scale words lie in one 16-byte piece of the tile.

#include "micro_common.cuh"

namespace b2g {
namespace micro {

constexpr int kWarps = 8;  // per block
constexpr int64_t kOneBlock = 16384;  // chunks of eight values up to which one block finds the tensor scale

// ---------------------------------------------------------------- largest magnitude -> NVFP4 tensor scale
// The smallest power of two 2^e >= 2^-100 with amax <= 2688 * 2^e (2688 = 6 * 448 = 1.3125 * 2^11). Every block takes
// the maximum of its own candidate: the order does not matter. Infinities and NaN do not count. Up to kOneBlock chunks
// one block does it alone, without a launch that clears the scale first (16x4096: 3 us less). 4096x14336 takes 24 us,
// three of them the launch that clears the scale: reading alone takes 21 (5.6 TB/s), and no other launch shape (256 to 1024
// threads a block, two to eight loads in flight each, 296 to 7104 blocks) was faster.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t a = __float_as_uint(v) & 0x7fffffffu;
  return a >= 0x7f800000u ? 0u : a;
}

// amax8 of the finite ones
template <typename T>
__device__ __forceinline__ uint32_t finite_amax8(const Raw8<T>& r) {
  const uint32_t a = amax8(r);
  if (a < 0x7f800000u) return a;
  float v[8];
  unpack8(r, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i]));
  return m;
}

// FLAT: rows follow one another without a gap, and are one row of `cols` values in `chunks` whole chunks and a rest.
// Else a row's eight-column chunks are numbered across rows; a thread steps by the whole grid, four chunks in flight,
// and carries (row, chunk) along instead of dividing.
template <typename T, int MODE, bool FLAT>
__global__ void __launch_bounds__(1024)
    tensor_scale_kernel(Mat x, int64_t rows, int64_t cols, int64_t chunks, int64_t step_rows, int64_t step_chunks, float* scale) {
  const int64_t first = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  int64_t row = FLAT ? 0 : first / chunks, k = FLAT ? first : first - row * chunks;
  const T* p = static_cast<const T*>(x.p);
  uint32_t m = 0;
  if constexpr (FLAT) {
    constexpr int U = sizeof(T) == 4 ? 4 : 8;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (k = first; k < chunks; k += U * step) {
      Raw8<T> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = load8<T, kVec>(p, 1, (k + u * step) * 8, chunks * 8, nullptr);
#pragma unroll
      for (int u = 0; u < U; ++u) m = max(m, finite_amax8(r[u]));
    }
    if (first < cols - chunks * 8) m = max(m, finite_bits(to_f32(p[chunks * 8 + first])));  // the last, fewer than eight
  } else {
    while (row < rows) {
      Raw8<T> r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        r[u] = load8<T, MODE>(p + row * x.sr, x.sc, k * 8, row < rows ? cols : 0, nullptr);
        row += step_rows;
        k += step_chunks;
        if (k >= chunks) {
          k -= chunks;
          ++row;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) m = max(m, finite_amax8(r[u]));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t part[32];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = __reduce_max_sync(0xffffffffu, threadIdx.x < blockDim.x / 32 ? part[threadIdx.x] : 0u);
    const int e = max(static_cast<int>(m >> 23) - 11 + ((m & 0x7fffffu) > 0x280000u ? 1 : 0), 27) << 23;
    if (threadIdx.x == 0) {
      if (gridDim.x == 1) *reinterpret_cast<int*>(scale) = e;
      else atomicMax(reinterpret_cast<int*>(scale), e);  // positive floats order as their bits do
    }
  }
}

// ---------------------------------------------------------------- rows -> codes and scales
// 4096x14336 bf16: mxfp8 31 us (5.7 TB/s), mxfp4 30, nvfp4 37; with the gate in front, 2048x14336: mxfp8 29 us (5.0 TB/s).
// The integer pipe is three quarters busy (unpacking, magnitudes, conversions): it and memory share the bound.
// Source of the rows' values: the values themselves, or the gate of a [gate | up] row.
template <typename T>
struct ValueSource {
  static constexpr int kLoads = 1;
  static constexpr bool kExact = true;
  __device__ __forceinline__ static uint32_t value(const Raw8<T> (&r)[1], float (&v)[8]) {  // and their amax8
    unpack8(r[0], v);
    return amax8(r[0]);
  }
};

// 1 / (1 + exp(-x)) and 1 / (1 + exp(x)) from e = exp(-|x|), which is at most one: nothing overflows, and both keep their
// digits however small they are. Exponential and division are the fast forms: their errors (2 + 1.173 |x| and 2 ulps)
// are below the rounding of any output type.
__device__ __forceinline__ float2 sigmoids(float x) {
  const float e = __expf(-fabsf(x)), inv = __fdividef(1.f, 1.f + e);
  return x >= 0.f ? make_float2(inv, e * inv) : make_float2(e * inv, inv);
}

template <typename T>
struct GateSource {
  static constexpr int kLoads = 2;
  static constexpr bool kExact = false;
  __device__ __forceinline__ static uint32_t value(const Raw8<T> (&r)[2], float (&v)[8]) {
    float g[8], u[8];
    unpack8(r[0], g);
    unpack8(r[1], u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = g[i] * sigmoids(g[i]).x * u[i];
    return amax8(v);
  }
};

template <typename T, int FMT, int MODE, template <typename> class SRC>
__global__ void __launch_bounds__(kWarps * 32)
    quantize_rows_kernel(Mat x, int64_t rows, int64_t cols, Quant q, int64_t col_chunks, int64_t tasks) {
  const int lane = threadIdx.x & 31;
  const int64_t task = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  // neighbouring warps take neighbouring column chunks of the same rows
  const int64_t rj = task / col_chunks;
  const int64_t c = (task - rj * col_chunks) * 256 + lane * 8;
  const int64_t row0 = (rj >> 5) * 128 + (rj & 31);
  CodePlace<FMT> to(q, row0, c, lane);  // of the first row; row i is 32 i rows and 4 i scale bytes on
  const int64_t code_step = 32 * q.pitch;
  const int live = row0 >= rows ? 0 : static_cast<int>(min(static_cast<int64_t>(4), (rows - row0 + 31) / 32));
  using S = SRC<T>;
  T* scratch = warp_scratch<T, MODE, kWarps>();
  Frag<T, MODE> f[4][S::kLoads];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int k = 0; k < S::kLoads; ++k)
      f[i][k] = fetch8<T, MODE>(static_cast<const T*>(x.p) + (row0 + 32 * i) * x.sr + k * cols * x.sc, x.sc, c, i < live ? cols : 0);
  }
  const TensorScale ts(FMT == FMT_NVFP4 ? *q.scale : 1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < live) {
      Raw8<T> r[S::kLoads];
#pragma unroll
      for (int k = 0; k < S::kLoads; ++k) r[k] = settle8<T, MODE>(f[i][k], scratch);
      float v[8];
      const uint32_t m = S::value(r, v);
      quantize_store<FMT, S::kExact>(v, m, lane, to, ts);
    } else if (to.leads) {  // a row past the last: zero scales and no codes
      *reinterpret_cast<uint32_t*>(to.word) = 0u;
    }
    to.codes += code_step;
    to.word += 4;
  }
}

// ---------------------------------------------------------------- columns (a transposed view) -> codes and scales
// x has unit ROW stride: what is contiguous in memory runs along the rows of the tensor that is made, across blocks.
// A block takes 128 rows x 128 columns; a lane holds 4 rows x 32 columns in registers (32 loads of 4 values, a warp's
// load covering 128 consecutive values), finds its rows' largest magnitudes without any exchange, and leaves codes in
// shared memory, from which whole rows of the tile are stored. Four warps, 32 columns each. mxfp8 of a transposed
// 4096x14336 bf16 matrix 36 us (4.9 TB/s), of 2047x4096 6.6 us; registers (128 a thread) and the integer pipe bound it.
template <typename T>
struct Raw4 {
  uint2 v;
};
template <>
struct Raw4<float> {
  uint4 v;
};

template <typename T>
__device__ __forceinline__ void unpack4(const Raw4<T>& r, float (&o)[4]) {
  const float2 a = pair_f32(r.v.x, static_cast<T*>(nullptr)), b = pair_f32(r.v.y, static_cast<T*>(nullptr));
  o[0] = a.x;
  o[1] = a.y;
  o[2] = b.x;
  o[3] = b.y;
}
__device__ __forceinline__ void unpack4(const Raw4<float>& r, float (&o)[4]) {
  o[0] = __uint_as_float(r.v.x);
  o[1] = __uint_as_float(r.v.y);
  o[2] = __uint_as_float(r.v.z);
  o[3] = __uint_as_float(r.v.w);
}

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(128) quantize_cols_kernel(Mat x, int64_t rows, int64_t cols, Quant q) {
  constexpr int kRowBytes = FMT == FMT_MXFP8 ? 128 : 64;       // a tile row's codes
  constexpr int kPieces = kRowBytes / 16;                      // in 16-byte pieces
  constexpr int kWarpPieces = kPieces / 4;                     // of one warp's 32 columns: 2 or 1
  constexpr int kBlk = block_of(FMT), kSub = 32 / kBlk;        // blocks in a warp's 32 columns: 1 or 2
  constexpr int kScaleBytes = 128 * 4 * kSub;                  // the tile's scales: 1 or 2 tiles of 512 bytes
  __shared__ uint4 codes[128 * kPieces];
  __shared__ __align__(16) uint8_t scales[kScaleBytes];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rt = blockIdx.x;                               // row tile
  const int64_t ct = blockIdx.y;                               // 128-column tile
  const int64_t r0 = rt * 128 + lane * 4, c0 = ct * 128 + warp * 32;
  const T* p = static_cast<const T*>(x.p);
  Raw4<T> raw[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int64_t c = c0 + i;
    const T* at = p + r0 + c * x.sc;
    if (VEC && c < cols && r0 + 4 <= rows) {
      raw[i].v = __ldg(reinterpret_cast<const decltype(raw[i].v)*>(at));
    } else {
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = c < cols && r0 + k < rows ? to_f32(at[k]) : 0.f;
      if constexpr (sizeof(T) == 4) {
        raw[i].v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      } else {
        raw[i].v = make_uint2(pack_pair(f[0], f[1], static_cast<T*>(nullptr)), pack_pair(f[2], f[3], static_cast<T*>(nullptr)));
      }
    }
  }
  const TensorScale ts(FMT == FMT_NVFP4 ? *q.scale : 1.f);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = lane * 4 + k;  // tile row
    uint32_t word[8];            // 32 columns' codes: 8 words (e4m3) or 4 (e2m1)
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      float v[kBlk];
      float m = 0.f, bad = 0.f;  // as amax8 of values
#pragma unroll
      for (int i = 0; i < kBlk; ++i) {
        float f[4];
        unpack4(raw[s * kBlk + i], f);
        v[i] = f[k];
        m = fmaxf(m, fabsf(v[i]));
        bad = fmaf(v[i], 0.f, bad);
      }
      BlockQuant<FMT> b;
      b.init(bad == 0.f ? __float_as_uint(m) : 0x7fffffffu, ts);
#pragma unroll
      for (int g = 0; g < kBlk / 8; ++g) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = v[8 * g + i];
        const uint2 w = codes8<FMT, true>(e, b);
        if constexpr (FMT == FMT_MXFP8) {
          word[2 * g] = w.x;
          word[2 * g + 1] = w.y;
        } else {
          word[s * (kBlk / 8) + g] = w.x;
        }
      }
      const int blk = warp * kSub + s;  // block of the tile's 4 or 8
      scales[(blk >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (blk & 3)] = static_cast<uint8_t>(b.byte);
    }
#pragma unroll
    for (int h = 0; h < kWarpPieces; ++h)  // pieces XOR-ed by the row so that a warp's stores spread over the banks
      codes[r * kPieces + ((warp * kWarpPieces + h) ^ ((r >> 2) & (kPieces - 1)))] =
          make_uint4(word[4 * h], word[4 * h + 1], word[4 * h + 2], word[4 * h + 3]);
  }
  __syncthreads();
  const int64_t code_bytes = FMT == FMT_MXFP8 ? q.code_cols : q.code_cols / 2;
  for (int i = threadIdx.x; i < 128 * kPieces; i += 128) {
    const int r = i / kPieces, h = i % kPieces;
    const int64_t at = ct * kRowBytes + h * 16;
    if (rt * 128 + r < rows && at < code_bytes)
      *reinterpret_cast<uint4*>(q.codes + (rt * 128 + r) * q.pitch + at) = codes[r * kPieces + (h ^ ((r >> 2) & (kPieces - 1)))];
  }
  if (threadIdx.x < kScaleBytes / 16) {
    const int64_t kt = ct * kSub + threadIdx.x / 32;
    if (kt < q.ktiles)
      *reinterpret_cast<uint4*>(q.scales + (rt * q.ktiles + kt) * 512 + (threadIdx.x & 31) * 16) =
          reinterpret_cast<const uint4*>(scales)[threadIdx.x];
  }
}

// ---------------------------------------------------------------- codes and scales -> values
// Bound by memory: 4096x14336 to bf16 from mxfp8 29 us (6.1 TB/s), from nvfp4 26 us (5.8 TB/s).
// A lane reads eight columns' codes of four rows, twice (256 columns apart), with each block's one scale byte, and
// stores 16 bytes a row (fp32: 32), a warp 512 consecutive ones.
template <typename T, int FMT, int MODE>
__global__ void __launch_bounds__(kWarps * 32)
    dequantize_kernel(const uint8_t* codes, int64_t pitch, const uint8_t* scales, const float* scale, int64_t rows,
                      int64_t cols, int64_t ktiles, T* out, int64_t sr, int64_t sc, int64_t col_chunks, int64_t tasks) {
  const int lane = threadIdx.x & 31;
  const int64_t task = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const int64_t rj = task / col_chunks;
  const int64_t c0 = (task - rj * col_chunks) * 512 + lane * 8;
  const int64_t row0 = (rj >> 5) * 128 + (rj & 31);
  const float ts = FMT == FMT_NVFP4 ? *scale : 1.f;
  T* scratch = warp_scratch<T, MODE, kWarps>();
  uint2 q[2][4];
  uint32_t s[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t c = c0 + 256 * h, blk = c / block_of(FMT);
    const uint8_t* sp = scales + scale_row(row0, ktiles) + (blk >> 2) * 512 + (blk & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + 32 * i;
      q[h][i] = make_uint2(0u, 0u);
      s[h][i] = 0u;
      if (row < rows && c < cols) {  // a row's codes are readable up to a multiple of 32 columns
        if constexpr (FMT == FMT_MXFP8) q[h][i] = __ldg(reinterpret_cast<const uint2*>(codes + row * pitch + c));
        else q[h][i].x = __ldg(reinterpret_cast<const uint32_t*>(codes + row * pitch + (c >> 1)));
        s[h][i] = __ldg(sp + i * 4);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t c = c0 + 256 * h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + 32 * i;
      if (row >= rows || c - lane * 8 >= cols) break;
      float bs;
      if constexpr (FMT == FMT_NVFP4) bs = e4m3_to_f32(s[h][i]);
      else bs = mx_scale_value(s[h][i]);
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        __half2_raw p;
        if constexpr (FMT == FMT_MXFP8)
          p = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((k < 2 ? q[h][i].x : q[h][i].y) >> (16 * (k & 1))), __NV_E4M3);
        else
          p = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(q[h][i].x >> (8 * k)), __NV_E2M1);
        const float2 f = __half22float2(__half2(p));
        // code * block scale is exact in fp32 (4 bits of e4m3 with a power of two, 2 bits of e2m1 with 4 of e4m3)
        v[2 * k] = f.x * bs;
        v[2 * k + 1] = f.y * bs;
        if constexpr (FMT == FMT_NVFP4) {
          v[2 * k] *= ts;
          v[2 * k + 1] *= ts;
        }
      }
      store8<T, MODE>(out + row * sr, sc, c, cols, pack8<T>(v), scratch);
    }
  }
}

// ---------------------------------------------------------------- the gate as values, and its gradient
// Bound by memory: 2048x14336 28 us (6.4 TB/s), its gradient 44 us (6.6 TB/s).
template <typename T, int MODE>
__global__ void __launch_bounds__(256) gate_kernel(Mat x, T* y, int64_t syr, int64_t syc, int64_t rows, int64_t cols, uint32_t row_blocks) {
  // blockDim.y rows of blockDim.x chunks of eight columns (kUnit: whole warps of them); row_blocks blocks along a row
  const uint32_t k = blockIdx.x % row_blocks * blockDim.x + threadIdx.x;
  const int64_t row = static_cast<int64_t>(blockIdx.x / row_blocks) * blockDim.y + threadIdx.y, c = static_cast<int64_t>(k) * 8;
  if (row >= rows || (MODE == kUnit ? c - (threadIdx.x & 31) * 8 : c) >= cols) return;
  T* scratch = warp_scratch<T, MODE, 8>();
  const T* p = static_cast<const T*>(x.p) + row * x.sr;
  const Frag<T, MODE> f = fetch8<T, MODE>(p, x.sc, c, cols), g = fetch8<T, MODE>(p + cols * x.sc, x.sc, c, cols);
  const Raw8<T> r[2] = {settle8<T, MODE>(f, scratch), settle8<T, MODE>(g, scratch)};
  float v[8];
  GateSource<T>::value(r, v);
  store8<T, MODE>(y + row * syr, syc, c, cols, pack8<T>(v), scratch);
}

// With s = sigmoid(g): d up = dy * (g s), d gate = dy * up * (s + g s (1 - s)). 1 - s is taken as sigmoid(-g), which keeps
// its digits where s is near one. bf16's dy * up may leave fp32's range where the gradient does not (a mask's lowest values,
// a small s), and so may the factor times the smaller of them: half the factor meets the larger one first.
template <typename T>
__device__ __forceinline__ void gate_gradient(float g, float u, float d, float& dg, float& du) {
  const float2 s = sigmoids(g);
  const float gs = g * s.x, factor = fmaf(gs, s.y, s.x);
  du = d * gs;
  if constexpr (std::is_same<T, __half>::value) {
    dg = d * u * factor;
  } else {
    float larger;  // of dy's and up's magnitudes, with the product's sign
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(larger) : "f"(d), "f"(u));
    dg = 0.5f * factor * larger * fminf(fabsf(d), fabsf(u)) * 2.f;
  }
}

// Aligned rows take 32 registers a thread, so that SMs are full.
template <typename T, int MODE>
__global__ void __launch_bounds__(256, MODE == kVec ? 8 : 0)
    gate_backward_kernel(Mat dy, Mat x, T* dx, int64_t sxr, int64_t sxc, int64_t rows, int64_t cols,
                         uint32_t row_blocks) {
  // blockDim.y rows of blockDim.x chunks of eight columns (kUnit: whole warps of them); row_blocks blocks along a row
  const uint32_t k = blockIdx.x % row_blocks * blockDim.x + threadIdx.x;
  const int64_t row = static_cast<int64_t>(blockIdx.x / row_blocks) * blockDim.y + threadIdx.y, c = static_cast<int64_t>(k) * 8;
  if (row >= rows || (MODE == kUnit ? c - (threadIdx.x & 31) * 8 : c) >= cols) return;
  T* scratch = warp_scratch<T, MODE, 8>();
  const T* p = static_cast<const T*>(x.p) + row * x.sr;
  const Frag<T, MODE> fg = fetch8<T, MODE>(p, x.sc, c, cols), fu = fetch8<T, MODE>(p + cols * x.sc, x.sc, c, cols);
  const Frag<T, MODE> fd = fetch8<T, MODE>(static_cast<const T*>(dy.p) + row * dy.sr, dy.sc, c, cols);
  const Raw8<T> rg = settle8<T, MODE>(fg, scratch), ru = settle8<T, MODE>(fu, scratch), rd = settle8<T, MODE>(fd, scratch);
  float g[8], u[8], d[8], dg[8], du[8];
  unpack8(rg, g);
  unpack8(ru, u);
  unpack8(rd, d);
#pragma unroll
  for (int i = 0; i < 8; ++i) gate_gradient<T>(g[i], u[i], d[i], dg[i], du[i]);
  T* o = dx + row * sxr;
  store8<T, MODE>(o, sxc, c, cols, pack8<T>(dg), scratch);
  store8<T, MODE>(o + cols * sxc, sxc, c, cols, pack8<T>(du), scratch);
}

// ---------------------------------------------------------------- host side
// Blocks of 256 threads over rows of eight-column chunks: several rows a block where they are short. Chunks are counted in
// 32 bits, the last block's included: rows of more are given a grid past every limit.
struct RowBlocks {
  dim3 block;
  uint32_t along;
  int64_t grid;
};

RowBlocks row_blocks(int64_t rows, int64_t cols, int mode) {
  const int64_t chunks = ceil_div(cols, 8);
  unsigned x = mode == kUnit ? 32 : 1;
  while (x < chunks && x < 256) x *= 2;
  RowBlocks b{dim3(x, 256 / x), static_cast<uint32_t>(ceil_div(chunks, x)), 0};
  b.grid = chunks > (int64_t(1) << 32) - 256 ? kMaxGrid + 1 : ceil_div(rows, b.block.y) * b.along;
  return b;
}

template <typename T, int FMT, int MODE, template <typename> class SRC>
int32_t run_rows(const Mat& x, int64_t rows, int64_t cols, const Quant& q, cudaStream_t st) {
  const int64_t col_chunks = ceil_div(q.ktiles * 4 * block_of(FMT), 256);  // whole scale tiles, so that all are written
  const int64_t tasks = ceil_div(rows, 128) * 32 * col_chunks;
  const int64_t grid = ceil_div(tasks, kWarps);
  if (grid > kMaxGrid) return too_large("quantisation");
  quantize_rows_kernel<T, FMT, MODE, SRC><<<static_cast<unsigned>(grid), kWarps * 32, 0, st>>>(x, rows, cols, q, col_chunks, tasks);
  return launched("quantize launch");
}

template <typename T, int FMT>
int32_t run_quantize(const b2g_micro_matrix* x, const b2g_micro_tensor* t, cudaStream_t st) {
  const Quant q = quant(t);
  const Mat m = mat(x);
  // Contiguous along the rows and not along the columns: the transposed kernel (4096 x 2047 bf16 through its transpose
  // takes it from the strided loads of the other). One column is read alike by both.
  if (x->stride_r == 1 && x->stride_c != 1 && t->cols > 1 && t->rows > 1) {
    const int64_t gx = ceil_div(t->rows, 128), gy = ceil_div(t->cols, 128);
    if (gy <= 65535) {
      const bool vec = (reinterpret_cast<uintptr_t>(x->ptr) % (4 * sizeof(T))) == 0 && x->stride_c % 4 == 0;
      const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
      if (vec) quantize_cols_kernel<T, FMT, true><<<grid, 128, 0, st>>>(m, t->rows, t->cols, q);
      else quantize_cols_kernel<T, FMT, false><<<grid, 128, 0, st>>>(m, t->rows, t->cols, q);
      return launched("quantize launch");
    }
  }
  return by_mode(mode_of(x, t->rows, t->cols, sizeof(T)), [&](auto mode) {
    return run_rows<T, FMT, decltype(mode)::value, ValueSource>(m, t->rows, t->cols, q, st);
  });
}

}  // namespace micro
}  // namespace b2g

using namespace b2g;
using namespace b2g::micro;

extern "C" {

int32_t b2g_micro_layout(int32_t format, int64_t rows, int64_t cols, int64_t* pitch, int64_t* scale_bytes) {
  return guarded([&]() -> int32_t {
    if (format < FMT_MXFP8 || format > FMT_NVFP4 || rows < 0 || cols < 0 || !pitch || !scale_bytes)
      return record_error(B2G_ERR_INVALID_ARG, "layout: bad format, dimension or output pointer");
    *pitch = min_pitch(format, cols);
    *scale_bytes = ceil_div(rows, 128) * ceil_div(cols, 4 * block_of(format)) * 512;
    return B2G_OK;
  });
}

int32_t b2g_micro_tensor_scale(const b2g_micro_matrix* x, int64_t rows, int64_t cols, int32_t dtype, float* scale,
                               void* stream) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || dtype < B2G_VALUE_F16 || dtype > B2G_VALUE_F32 || !scale)
      return record_error(B2G_ERR_INVALID_ARG, "tensor_scale: bad dimension, dtype or output pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows && cols)
      if (const int32_t rc = check_matrix(x, "x")) return rc;
    const b2g_micro_matrix none = {nullptr, 0, 1};
    if (!rows || !cols) x = &none;
    return by_type(dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      Mat m = mat(x);
      int64_t r = rows, c = cols;
      if (x->stride_r == 1 && x->stride_c != 1) {  // the maximum does not care which way the matrix lies
        std::swap(m.sr, m.sc);
        std::swap(r, c);
      }
      const b2g_micro_matrix view = {const_cast<void*>(m.p), m.sr, m.sc};
      if (!rows || !cols) {  // no values: one flat row of no chunks, nothing is read
        r = 1;
        c = 0;
      }
      const int64_t chunks = ceil_div(c, 8);
      unsigned threads = 1024, grid = 1;
      if (r * chunks > kOneBlock) {
        const int64_t want = ceil_div(r * chunks, kWarps * 32 * 4);
        threads = kWarps * 32;
        grid = static_cast<unsigned>(want > 148 * 8 ? 148 * 8 : want);
        const cudaError_t e = cudaMemsetAsync(scale, 0, sizeof(float), st);
        if (e != cudaSuccess) {
          cudaGetLastError();
          return record_error(B2G_ERR_CUDA, std::string("memset: ") + cudaGetErrorString(e));
        }
      }
      const int64_t step = static_cast<int64_t>(grid) * threads;
      if (m.sc == 1 && aligned16(m.p) && (r == 1 || m.sr == c))
        tensor_scale_kernel<T, kVec, true><<<grid, threads, 0, st>>>(m, 1, r * c, r * c / 8, 0, 0, scale);
      else if (mode_of(&view, r, c, sizeof(T)) == kVec)
        tensor_scale_kernel<T, kVec, false><<<grid, threads, 0, st>>>(m, r, c, chunks, step / chunks, step % chunks, scale);
      else
        tensor_scale_kernel<T, kAny, false><<<grid, threads, 0, st>>>(m, r, c, chunks, step / chunks, step % chunks, scale);
      return launched("tensor_scale launch");
    });
  });
}

int32_t b2g_micro_quantize(const b2g_micro_matrix* x, int32_t dtype, const b2g_micro_tensor* q, void* stream) {
  return guarded([&]() -> int32_t {
    if (const int32_t rc = check_tensor(q, "q")) return rc;
    if (dtype < B2G_VALUE_F16 || dtype > B2G_VALUE_F32) return record_error(B2G_ERR_INVALID_ARG, "quantize: bad dtype");
    if (q->rows == 0 || q->cols == 0) return B2G_OK;
    if (const int32_t rc = check_matrix(x, "x")) return rc;
    return by_type(dtype, [&](auto t) {
      return by_format(q->format, [&](auto f) {
        return run_quantize<decltype(t), decltype(f)::value>(x, q, static_cast<cudaStream_t>(stream));
      });
    });
  });
}

int32_t b2g_micro_dequantize(const b2g_micro_tensor* q, const b2g_micro_matrix* out, int32_t dtype, void* stream) {
  return guarded([&]() -> int32_t {
    if (const int32_t rc = check_tensor(q, "q")) return rc;
    if (dtype < B2G_VALUE_F16 || dtype > B2G_VALUE_F32) return record_error(B2G_ERR_INVALID_ARG, "dequantize: bad dtype");
    if (q->rows == 0 || q->cols == 0) return B2G_OK;
    if (const int32_t rc = check_matrix(out, "out")) return rc;
    const int64_t col_chunks = ceil_div(q->cols, 512), tasks = ceil_div(q->rows, 128) * 32 * col_chunks;
    const int64_t grid = ceil_div(tasks, kWarps);
    if (grid > kMaxGrid) return too_large("dequantisation");
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      return by_format(q->format, [&](auto f) -> int32_t {
        constexpr int F = decltype(f)::value;
        const auto go = [&](auto kernel) {
          kernel<<<static_cast<unsigned>(grid), kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(
              static_cast<const uint8_t*>(q->codes), q->pitch, static_cast<const uint8_t*>(q->scales), q->scale, q->rows,
              q->cols, ceil_div(q->cols, 4 * block_of(F)), static_cast<T*>(out->ptr), out->stride_r, out->stride_c,
              col_chunks, tasks);
        };
        return by_mode(mode_of(out, q->rows, q->cols, sizeof(T)), [&](auto mode) {
          go(dequantize_kernel<T, F, decltype(mode)::value>);
          return launched("dequantize launch");
        });
      });
    });
  });
}

int32_t b2g_micro_silu_mul(const b2g_micro_matrix* gate_up, const b2g_micro_matrix* y, const b2g_micro_tensor* q,
                           int64_t rows, int64_t cols, int32_t dtype, void* stream) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || (dtype != B2G_VALUE_F16 && dtype != B2G_VALUE_BF16) || (!y && !q) || (y && q))
      return record_error(B2G_ERR_INVALID_ARG, "silu_mul: bad dimension or dtype, or not one output");
    if (q) {
      if (const int32_t rc = check_tensor(q, "q")) return rc;
      if (q->rows != rows || q->cols != cols) return record_error(B2G_ERR_INVALID_ARG, "silu_mul: q is not [rows, cols]");
    }
    if (rows == 0 || cols == 0) return B2G_OK;
    if (const int32_t rc = check_matrix(gate_up, "gate_up")) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_type(dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      if constexpr (sizeof(T) == 4) {
        return B2G_ERR_INVALID_ARG;
      } else {
        int mode = mode_of(gate_up, rows, cols, 2);  // kVec: the up half, `cols` values into the row, is aligned too
        if (q) {
          return by_format(q->format, [&](auto f) {
            return by_mode(mode, [&](auto md) {
              return run_rows<T, decltype(f)::value, decltype(md)::value, GateSource>(mat(gate_up), rows, cols, quant(q), st);
            });
          });
        }
        if (const int32_t rc = check_matrix(y, "y")) return rc;
        mode = std::max(mode, mode_of(y, rows, cols, 2));
        const RowBlocks rb = row_blocks(rows, cols, mode);
        if (rb.grid > kMaxGrid) return too_large("silu_mul");
        by_mode(mode, [&](auto md) -> int32_t {
          gate_kernel<T, decltype(md)::value><<<static_cast<unsigned>(rb.grid), rb.block, 0, st>>>(
              mat(gate_up), static_cast<T*>(y->ptr), y->stride_r, y->stride_c, rows, cols, rb.along);
          return B2G_OK;
        });
        return launched("silu_mul launch");
      }
    });
  });
}

int32_t b2g_micro_silu_mul_backward(const b2g_micro_matrix* dy, const b2g_micro_matrix* gate_up,
                                    const b2g_micro_matrix* dgate_up, int64_t rows, int64_t cols, int32_t dtype,
                                    void* stream) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || (dtype != B2G_VALUE_F16 && dtype != B2G_VALUE_BF16))
      return record_error(B2G_ERR_INVALID_ARG, "silu_mul_backward: bad dimension or dtype");
    if (rows == 0 || cols == 0) return B2G_OK;
    if (const int32_t rc = check_matrix(dy, "dy")) return rc;
    if (const int32_t rc = check_matrix(gate_up, "gate_up")) return rc;
    if (const int32_t rc = check_matrix(dgate_up, "dgate_up")) return rc;
    return by_type(dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      if constexpr (sizeof(T) == 4) {
        return B2G_ERR_INVALID_ARG;
      } else {
        const int mode = std::max({mode_of(dy, rows, cols, 2), mode_of(gate_up, rows, cols, 2), mode_of(dgate_up, rows, cols, 2)});
        const RowBlocks rb = row_blocks(rows, cols, mode);
        if (rb.grid > kMaxGrid) return too_large("silu_mul_backward");
        by_mode(mode, [&](auto md) -> int32_t {
          gate_backward_kernel<T, decltype(md)::value><<<static_cast<unsigned>(rb.grid), rb.block, 0, static_cast<cudaStream_t>(stream)>>>(
              mat(dy), mat(gate_up), static_cast<T*>(dgate_up->ptr), dgate_up->stride_r, dgate_up->stride_c, rows, cols, rb.along);
          return B2G_OK;
        });
        return launched("silu_mul_backward launch");
      }
    });
  });
}

}  // extern "C"

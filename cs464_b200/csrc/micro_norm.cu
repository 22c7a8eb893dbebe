// micro_norm.cu — root-mean-square norm of a row with the residual's addition, its output as values or as a
// microscaled tensor, and its gradient.
//
// Bound by memory: each row is read once, held in registers between the sum of squares and the scaling, and written
// once. `tpr` threads share a row, eight consecutive columns each per round of tpr * 8 columns; ROUNDS rounds are held
// in registers (1, 2 or 4: as few as the row needs, since registers are what limits the rows in flight); past 4 rounds
// the row is read again (from L2). 8192x4096 bf16 with a residual: values 42 us (6.4 TB/s), mxfp8 45 us (5.2 TB/s, the
// integer pipe two thirds busy with the quantisation), the gradient 50 us (5.4 TB/s).

#include "micro_common.cuh"

namespace b2g {
namespace micro {

constexpr int kMostRounds = 4;
constexpr int kMaxThreads = 512;  // per row, and per block where that is more than 128
constexpr int64_t kMostCols = (int64_t(1) << 31) - 8192;

// Blocks of kMaxThreads an SM holds at once, by rounds held in registers.
constexpr int blocks_per_sm(int rounds) { return rounds <= 2 ? 2 : 1; }

constexpr int backward_blocks_per_sm(int rounds) { return rounds == 1 ? 2 : 1; }

// Sum over the `tpr` threads of each row of the block (tpr a multiple of 32; rows of a block are consecutive groups of
// warps), the same bits in every thread: warps by shuffles, then the row's warps in order through `part` (one float2
// per warp). `buf` alternates so that one barrier per call is enough.
__device__ __forceinline__ float2 row_sum(float2 v, int tpr, float2 (*part)[32], int buf) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, d);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
  }
  if (tpr == 32) return v;
  const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp / per * per;
  if ((threadIdx.x & 31) == 0) part[buf][warp] = v;
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int i = 0; i < per; ++i) {
    s.x += part[buf][first + i].x;
    s.y += part[buf][first + i].y;
  }
  return s;
}

// FMT_NONE writes values (y), the formats write q; rows from `rows` to the end of their 128-row scale tile get zero
// scales. RES: h = x + residual, else h = x. Columns, counted on to the end of a round, fit 31 bits (kMostCols).
template <typename T, int FMT, bool RES, int MODE, int ROUNDS>
__global__ void __launch_bounds__(kMaxThreads, blocks_per_sm(ROUNDS))
    norm_kernel(Mat x, Mat res, const T* w, T* h, int64_t shr, int64_t shc, T* y, int64_t syr, int64_t syc, Quant q,
                int64_t rows, int cols, float eps, int tpr) {
  __shared__ float2 part[2][32];
  const int t = threadIdx.x % tpr;
  const int64_t row = blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < rows;
  const int width = tpr * 8;
  if (FMT != FMT_NONE && blockIdx.x * static_cast<int64_t>(blockDim.x / tpr) >= rows) {  // a block without rows
    for (int64_t kt = t; kt < q.ktiles; kt += tpr)
      *reinterpret_cast<uint32_t*>(q.scales + scale_row(row, q.ktiles) + kt * 512) = 0u;
    return;
  }
  const T* xr = static_cast<const T*>(x.p) + row * x.sr;
  const T* rr = RES ? static_cast<const T*>(res.p) + row * res.sr : nullptr;
  T* hr = h + row * shr;
  const int lim = live ? cols : 0;
  const TensorScale ts(FMT == FMT_NVFP4 ? *q.scale : 1.f);
  T* scratch = warp_scratch<T, MODE, kMaxThreads / 32>();
  const int lane8 = (threadIdx.x & 31) * 8;  // a lane's columns past its warp's first

  float2 s = make_float2(0.f, 0.f);
  // v = the row's values from their loads; stores h and adds up the squares
  auto take = [&](const Raw8<T>& a, const Raw8<T>& b, int c, float(&v)[8]) {
    unpack8(a, v);
    if (RES) {
      float f[8];
      unpack8(b, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += f[i];
      if (h) store8<T, MODE>(hr, shc, c, lim, pack8<T>(v), scratch);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s.x = fmaf(v[i], v[i], s.x);
  };
  float v[ROUNDS][8];
  {
    Frag<T, MODE> a[ROUNDS], b[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int c = k * width + t * 8;
      a[k] = fetch8<T, MODE>(xr, x.sc, c, lim);
      if (RES) b[k] = fetch8<T, MODE>(rr, res.sc, c, lim);
    }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const Raw8<T> ra = settle8<T, MODE>(a[k], scratch);
      take(ra, RES ? settle8<T, MODE>(b[k], scratch) : ra, k * width + t * 8, v[k]);
    }
  }
  if constexpr (ROUNDS == kMostRounds) {
    for (int64_t c = ROUNDS * width + t * 8; c - t * 8 < cols; c += width) {
      const Raw8<T> a = load8<T, MODE>(xr, x.sc, c, lim, scratch);
      Raw8<T> b = a;
      if (RES) b = load8<T, MODE>(rr, res.sc, c, lim, scratch);
      float f[8];
      take(a, b, static_cast<int>(c), f);
    }
  }
  s = row_sum(s, tpr, part, 0);
  const float r = rsqrtf(s.x / static_cast<float>(cols) + eps);

  const int64_t cover = FMT == FMT_NONE ? cols : q.ktiles * 4 * block_of(FMT);  // whole scale tiles
  auto finish = [&](float(&f)[8], int64_t c) {
    // Past the row's end values and weights are read as zero; a warp wholly past it has zeros whatever the row's norm
    // is.
    if (c - lane8 < lim) {
      float g[8];
      unpack8(load8<T, MODE>(w, 1, c, cols, scratch), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c < lim ? f[i] * r * g[i] : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    }
    if constexpr (FMT == FMT_NONE) {
      store8<T, MODE>(y + row * syr, syc, c, lim, pack8<T>(f), scratch);
    } else {
      CodePlace<FMT> to(q, row, c, threadIdx.x & 31);
      to.has_codes = to.has_codes && live;
      quantize_store<FMT, false>(f, amax8(f), threadIdx.x & 31, to, ts);
    }
  };
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k)
    if (k * width < cover) finish(v[k], k * width + t * 8);
  if constexpr (ROUNDS == kMostRounds) {
    for (int64_t c = ROUNDS * width + t * 8; c - t * 8 < cover; c += width) {
      float f[8];
      unpack8(load8<T, MODE>(xr, x.sc, c, lim, scratch), f);
      if (RES) {
        float g[8];
        unpack8(load8<T, MODE>(rr, res.sc, c, lim, scratch), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
      }
      finish(f, c);
    }
  }
}

// Gradient: a block walks rows, `rpb` groups of tpr threads a row each, so its threads keep their columns and add up
// the weight's gradient in registers (rounds past the fourth: in the block's own row of the workspace, from column
// ROUNDS * width on). At the end the block's groups add theirs up in shared memory, in order, and the block leaves one
// fp32 row in the workspace; norm_dweight_kernel adds the rows in a fixed order. With one or two rounds of aligned
// rows the weight stays in registers and a row's loads are one row ahead, in flight across the row sum's barrier; four
// leave no room for either.
template <typename T, bool DH, int MODE, int ROUNDS>
__global__ void __launch_bounds__(kMaxThreads, backward_blocks_per_sm(ROUNDS))
    norm_backward_kernel(Mat dy, Mat h, const T* w, Mat dh, T* dx, int64_t sxr, int64_t sxc, float* partial,
                         int64_t rows, int cols, float eps, int tpr) {
  __shared__ float2 part[2][32];
  extern __shared__ float sums[];  // [rpb][cols] where rpb > 1
  constexpr bool kAhead = MODE == kVec && ROUNDS < kMostRounds;
  T* scratch = warp_scratch<T, MODE, kMaxThreads / 32>();
  const int t = threadIdx.x % tpr, g = threadIdx.x / tpr;
  const int rpb = blockDim.x / tpr;
  const int width = tpr * 8, lane8 = (threadIdx.x & 31) * 8;
  const float n = static_cast<float>(cols);
  float* mine = partial + blockIdx.x * static_cast<int64_t>(cols);
  float acc[ROUNDS][8];
  Raw8<T> wr[kAhead ? ROUNDS : 1];
  auto weight = [&](int k, float(&wt)[8]) {
    if constexpr (kAhead) unpack8(wr[k], wt);
    else unpack8(load8<T, MODE>(w, 1, k * width + t * 8, cols, scratch), wt);
  };
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if constexpr (kAhead) wr[k] = load8<T, MODE>(w, 1, k * width + t * 8, cols, scratch);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[k][i] = 0.f;
  }
  Frag<T, MODE> a[ROUNDS], b[ROUNDS], e[DH ? ROUNDS : 1];
  auto fetch = [&](int64_t row) {
    const int lim = row < rows ? cols : 0;
    const T* dyr = static_cast<const T*>(dy.p) + row * dy.sr;
    const T* hr = static_cast<const T*>(h.p) + row * h.sr;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int c = k * width + t * 8;
      a[k] = fetch8<T, MODE>(dyr, dy.sc, c, lim);
      b[k] = fetch8<T, MODE>(hr, h.sc, c, lim);
      if (DH) e[k] = fetch8<T, MODE>(static_cast<const T*>(dh.p) + row * dh.sr, dh.sc, c, lim);
    }
  };
  // dx, and the weight's terms into `sum`
  auto finish = [&](const Raw8<T>& rd, const Raw8<T>& rv, const Raw8<T>& re, const float(&wt)[8], int64_t row, int64_t c,
                    int lim, float r, float rm, float(&sum)[8]) {
    float d[8], v[8], o[8];
    unpack8(rd, d);
    unpack8(rv, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = fmaf(v[i], -rm, d[i] * wt[i] * r);
      sum[i] = fmaf(d[i] * v[i], r, sum[i]);
    }
    if (DH) {
      unpack8(re, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] += d[i];
    }
    store8<T, MODE>(dx + row * sxr, sxc, c, lim, pack8<T>(o), scratch);
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * rpb;
  const int64_t trips = (rows - static_cast<int64_t>(blockIdx.x) * rpb + step - 1) / step;  // the block's; at least one
  int64_t row = blockIdx.x * static_cast<int64_t>(rpb) + g;
  int buf = 0;
  if (kAhead) fetch(row);
  for (int64_t trip = 0; trip < trips; ++trip, row += step) {
    const int lim = row < rows ? cols : 0;  // every thread of the block reaches the barrier
    float2 s = make_float2(0.f, 0.f);
    auto add = [&](const Raw8<T>& rd, const Raw8<T>& rv, const float(&wt)[8]) {
      float d[8], v[8];
      unpack8(rd, d);
      unpack8(rv, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.x = fmaf(v[i], v[i], s.x);
        s.y = fmaf(d[i] * wt[i], v[i], s.y);
      }
    };
    if (!kAhead) fetch(row);
    Raw8<T> ca[ROUNDS], cb[ROUNDS], ce[DH ? ROUNDS : 1];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      ca[k] = settle8<T, MODE>(a[k], scratch);
      cb[k] = settle8<T, MODE>(b[k], scratch);
      if (DH) ce[k] = settle8<T, MODE>(e[k], scratch);
      float wt[8];
      weight(k, wt);
      add(ca[k], cb[k], wt);
    }
    const T* dyr = static_cast<const T*>(dy.p) + row * dy.sr;
    const T* hr = static_cast<const T*>(h.p) + row * h.sr;
    if constexpr (ROUNDS == kMostRounds) {
      for (int64_t c = ROUNDS * width + t * 8; c - t * 8 < cols; c += width) {
        float wt[8];
        unpack8(load8<T, MODE>(w, 1, c, cols, scratch), wt);
        const Raw8<T> rd = load8<T, MODE>(dyr, dy.sc, c, lim, scratch);
        add(rd, load8<T, MODE>(hr, h.sc, c, lim, scratch), wt);
      }
    }
    if (kAhead && trip + 1 < trips) fetch(row + step);
    s = row_sum(s, tpr, part, buf);
    buf ^= 1;
    const float r = rsqrtf(s.x / n + eps);
    const float rm = s.y / n * r * r * r;  // dx = r * dy * w - h * rm; r^3 alone may leave fp32's range where rm does not
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const int c = k * width + t * 8;
      if (c - lane8 < lim) {
        float wt[8];
        weight(k, wt);
        finish(ca[k], cb[k], ce[DH ? k : 0], wt, row, c, lim, r, rm, acc[k]);
      }
    }
    if constexpr (ROUNDS == kMostRounds) {  // such rows are long: one group a block, whose columns are this thread's own
      for (int64_t c = ROUNDS * width + t * 8; c - lane8 < lim; c += width) {
        float wt[8], sum[8];
        unpack8(load8<T, MODE>(w, 1, c, cols, scratch), wt);
        const Raw8<T> rd = load8<T, MODE>(dyr, dy.sc, c, lim, scratch), rv = load8<T, MODE>(hr, h.sc, c, lim, scratch);
        Raw8<T> re = rd;
        if (DH) re = load8<T, MODE>(static_cast<const T*>(dh.p) + row * dh.sr, dh.sc, c, lim, scratch);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = trip > 0 && c + i < cols ? mine[c + i] : 0.f;
        finish(rd, rv, re, wt, row, c, lim, r, rm, sum);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < cols) mine[c + i] = sum[i];
      }
    }
  }
  if (rpb > 1) {
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k * width + t * 8 + i < cols) sums[g * cols + k * width + t * 8 + i] = acc[k][i];
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      float f = sums[c];
      for (int i = 1; i < rpb; ++i) f += sums[i * cols + c];
      mine[c] = f;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int c = k * width + t * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      if (c + i + 4 <= cols && cols % 4 == 0) {
        *reinterpret_cast<float4*>(mine + c + i) = make_float4(acc[k][i], acc[k][i + 1], acc[k][i + 2], acc[k][i + 3]);
      } else {
#pragma unroll
        for (int j = i; j < i + 4; ++j)
          if (c + j < cols) mine[c + j] = acc[k][j];
      }
    }
  }
}

// dweight[c] = sum over the blocks' partial rows: 32 strands, each its rows in order, then the strands in order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_dweight_kernel(const float* partial, int groups, int64_t cols, T* dw) {
  __shared__ float part[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * int64_t(32) + x;
  float s = 0.f;
  if (c < cols) {
    int g = y;
    for (; g + 96 < groups; g += 128) {
      float f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = partial[static_cast<int64_t>(g + 32 * u) * cols + c];
#pragma unroll
      for (int u = 0; u < 4; ++u) s += f[u];
    }
    for (; g < groups; g += 32) s += partial[static_cast<int64_t>(g) * cols + c];
  }
  part[y][x] = s;
  __syncthreads();
  if (y == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += part[i][x];
    dw[c] = from_f32<T>(s);
  }
}

struct Split {
  int tpr, threads, rounds;
  int64_t blocks, groups;
};

int pow2_threads(int64_t n, int most) {
  int t = 32;
  while (t < n && t < most) t *= 2;
  return t;
}

int rounds_of(int64_t cols, int tpr) {
  const int64_t n = ceil_div(cols, int64_t(tpr) * 8);
  return n <= 1 ? 1 : n <= 2 ? 2 : kMostRounds;
}

// Threads per row: with many rows, two rounds of eight columns a thread keep more loads in flight per thread; with
// few, one round shortens the row's own time. Blocks of at least 128 threads.
Split forward_split(int64_t rows, int64_t cols) {
  Split s;
  const int64_t chunks = ceil_div(cols, 8);
  s.tpr = rows >= 592 ? pow2_threads(ceil_div(chunks, 2), kMaxThreads) : pow2_threads(chunks, kMaxThreads);
  s.threads = s.tpr < 128 ? 128 : s.tpr;
  s.rounds = rounds_of(cols, s.tpr);
  s.groups = rows;
  s.blocks = ceil_div(rows, s.threads / s.tpr);
  return s;
}

// The gradient's blocks stay for many rows: as many as the GPU holds at once, fewer where there are fewer rows. Two
// rounds of eight columns a thread where there are that many; blocks of one row, or of 128 threads and several short
// rows.
Split backward_split(int64_t rows, int64_t cols) {
  Split s;
  s.tpr = pow2_threads(ceil_div(ceil_div(cols, 8), 2), kMaxThreads);
  s.threads = s.tpr < 128 ? 128 : s.tpr;
  s.rounds = rounds_of(cols, s.tpr);
  const int64_t most = 148 * backward_blocks_per_sm(s.rounds) * (kMaxThreads / s.threads);
  s.blocks = ceil_div(rows, s.threads / s.tpr);
  if (s.blocks > most) s.blocks = most;
  s.groups = s.blocks;
  return s;
}

}  // namespace micro
}  // namespace b2g

using namespace b2g;
using namespace b2g::micro;

extern "C" {

int32_t b2g_micro_rms_norm(const b2g_micro_matrix* x, const b2g_micro_matrix* residual, const void* weight,
                           const b2g_micro_matrix* h, const b2g_micro_matrix* y, const b2g_micro_tensor* q, int64_t rows,
                           int64_t cols, float eps, int32_t dtype, void* stream) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || (dtype != B2G_VALUE_F16 && dtype != B2G_VALUE_BF16) || (!y && !q) || (y && q))
      return record_error(B2G_ERR_INVALID_ARG, "rms_norm: bad dimension or dtype, or not one output");
    if (h && !residual) return record_error(B2G_ERR_INVALID_ARG, "rms_norm: without a residual h is x itself, pass NULL");
    if (q) {
      if (const int32_t rc = check_tensor(q, "q")) return rc;
      if (q->rows != rows || q->cols != cols) return record_error(B2G_ERR_INVALID_ARG, "rms_norm: q is not [rows, cols]");
    }
    if (cols > kMostCols) return too_large("rms_norm");
    if (rows == 0 || cols == 0) return B2G_OK;
    if (const int32_t rc = check_matrix(x, "x")) return rc;
    if (residual)
      if (const int32_t rc = check_matrix(residual, "residual")) return rc;
    if (h)
      if (const int32_t rc = check_matrix(h, "h")) return rc;
    if (y)
      if (const int32_t rc = check_matrix(y, "y")) return rc;
    if (!weight) return record_error(B2G_ERR_INVALID_ARG, "null weight");
    const Split s = forward_split(q ? ceil_div(rows, 128) * 128 : rows, cols);
    if (s.blocks > kMaxGrid) return too_large("rms_norm");
    const b2g_micro_matrix w = {const_cast<void*>(weight), cols, 1};
    int mode = std::max(mode_of(x, rows, cols, 2), mode_of(&w, 1, cols, 2));
    for (const b2g_micro_matrix* m : {residual, h, y})
      if (m) mode = std::max(mode, mode_of(m, rows, cols, 2));
    return by_type(dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      if constexpr (sizeof(T) == 4) {
        return B2G_ERR_INVALID_ARG;
      } else {
        const Mat none{nullptr, 0, 1};
        const auto go = [&](auto kernel) {
          kernel<<<static_cast<unsigned>(s.blocks), s.threads, 0, static_cast<cudaStream_t>(stream)>>>(
              mat(x), residual ? mat(residual) : none, static_cast<const T*>(weight), h ? static_cast<T*>(h->ptr) : nullptr,
              h ? h->stride_r : 0, h ? h->stride_c : 1, y ? static_cast<T*>(y->ptr) : nullptr, y ? y->stride_r : 0,
              y ? y->stride_c : 1, q ? quant(q) : Quant{}, rows, static_cast<int>(cols), eps, s.tpr);
          return launched("rms_norm launch");
        };
        const auto pick = [&](auto f) -> int32_t {
          constexpr int F = decltype(f)::value;
          return by_flag(residual, [&](auto res) {
            constexpr bool R = decltype(res)::value;
            if (mode == kAny) return go(norm_kernel<T, F, R, kAny, kMostRounds>);
            if (mode == kUnit) return s.rounds <= 2 ? go(norm_kernel<T, F, R, kUnit, 2>) : go(norm_kernel<T, F, R, kUnit, kMostRounds>);
            return s.rounds == 1   ? go(norm_kernel<T, F, R, kVec, 1>)
                   : s.rounds == 2 ? go(norm_kernel<T, F, R, kVec, 2>)
                                   : go(norm_kernel<T, F, R, kVec, kMostRounds>);
          });
        };
        return q ? by_format(q->format, pick) : pick(std::integral_constant<int, FMT_NONE>{});
      }
    });
  });
}

int32_t b2g_micro_rms_norm_workspace(int64_t rows, int64_t cols, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || !bytes) return record_error(B2G_ERR_INVALID_ARG, "rms_norm_workspace: bad argument");
    *bytes = rows && cols ? static_cast<size_t>(backward_split(rows, cols).groups * cols) * sizeof(float) : 0;
    return B2G_OK;
  });
}

int32_t b2g_micro_rms_norm_backward(const b2g_micro_matrix* dy, const b2g_micro_matrix* h, const void* weight,
                                    const b2g_micro_matrix* dh, const b2g_micro_matrix* dx, void* dweight,
                                    void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols, float eps,
                                    int32_t dtype, void* stream) {
  return guarded([&]() -> int32_t {
    if (rows < 0 || cols < 0 || (dtype != B2G_VALUE_F16 && dtype != B2G_VALUE_BF16))
      return record_error(B2G_ERR_INVALID_ARG, "rms_norm_backward: bad dimension or dtype");
    if (cols > kMostCols) return too_large("rms_norm_backward");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cols == 0) return B2G_OK;
    if (!dweight || !weight) return record_error(B2G_ERR_INVALID_ARG, "null weight or dweight");
    if (rows == 0) {  // a sum over no rows
      const cudaError_t e = cudaMemsetAsync(dweight, 0, static_cast<size_t>(cols) * 2, st);
      if (e == cudaSuccess) return B2G_OK;
      cudaGetLastError();
      return record_error(B2G_ERR_CUDA, std::string("memset: ") + cudaGetErrorString(e));
    }
    if (const int32_t rc = check_matrix(dy, "dy")) return rc;
    if (const int32_t rc = check_matrix(h, "h")) return rc;
    if (const int32_t rc = check_matrix(dx, "dx")) return rc;
    if (dh)
      if (const int32_t rc = check_matrix(dh, "dh")) return rc;
    const Split s = backward_split(rows, cols);
    if (!workspace || !aligned16(workspace) || workspace_bytes < static_cast<size_t>(s.groups * cols) * sizeof(float))
      return record_error(B2G_ERR_WORKSPACE, "rms_norm_backward: workspace missing, misaligned or too small");
    const int64_t wgrid = ceil_div(cols, 32);
    if (wgrid > kMaxGrid) return too_large("rms_norm_backward");
    const b2g_micro_matrix w = {const_cast<void*>(weight), cols, 1};
    int mode = std::max({mode_of(dy, rows, cols, 2), mode_of(h, rows, cols, 2), mode_of(dx, rows, cols, 2), mode_of(&w, 1, cols, 2)});
    if (dh) mode = std::max(mode, mode_of(dh, rows, cols, 2));
    return by_type(dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      if constexpr (sizeof(T) == 4) {
        return B2G_ERR_INVALID_ARG;
      } else {
        const Mat none{nullptr, 0, 1};
        const auto go = [&](auto kernel) {
          const size_t smem = s.threads > s.tpr ? size_t(s.threads / s.tpr) * cols * sizeof(float) : 0;
          kernel<<<static_cast<unsigned>(s.blocks), s.threads, smem, st>>>(
              mat(dy), mat(h), static_cast<const T*>(weight), dh ? mat(dh) : none, static_cast<T*>(dx->ptr), dx->stride_r,
              dx->stride_c, static_cast<float*>(workspace), rows, static_cast<int>(cols), eps, s.tpr);
          return launched("rms_norm_backward launch");
        };
        const int32_t rc = by_flag(dh, [&](auto f) {
          constexpr bool D = decltype(f)::value;
          if (mode == kAny) return go(norm_backward_kernel<T, D, kAny, kMostRounds>);
          if (mode == kUnit)
            return s.rounds <= 2 ? go(norm_backward_kernel<T, D, kUnit, 2>) : go(norm_backward_kernel<T, D, kUnit, kMostRounds>);
          return s.rounds == 1   ? go(norm_backward_kernel<T, D, kVec, 1>)
                 : s.rounds == 2 ? go(norm_backward_kernel<T, D, kVec, 2>)
                                 : go(norm_backward_kernel<T, D, kVec, kMostRounds>);
        });
        if (rc) return rc;
        norm_dweight_kernel<T><<<static_cast<unsigned>(wgrid), 1024, 0, st>>>(static_cast<const float*>(workspace),
                                                                           static_cast<int>(s.groups), cols,
                                                                           static_cast<T*>(dweight));
        return launched("rms_norm_backward reduce launch");
      }
    });
  });
}

}  // extern "C"

// micro_gemm.cu — products of two microscaled tensors on the block-scaled tensor-core kinds: C[M,N] = A[M,K] *
// B[N,K]^T.
//
// Both operands lie as codes with K contiguous and scales in the order the tensor core reads them, so nothing is
// converted on the way: TMA brings 128 bytes of codes a row (256 columns of 4 bits, 128 of 8) and the scale tiles that
// belong to them into a ring of shared-memory stages, tcgen05.cp moves the scales on into tensor memory (a region of
// its own for every stage, free once the stage's MMAs have completed), and four block-scaled MMAs of 32 bytes of K
// multiply the stage into fp32 accumulators. Two kernels:
//   product_kernel       one CTA per 128 x tile_q tile and K split; the MMA's 128 rows run over B's rows (a layer's
//                        weights), its narrow side over A's (the tokens), so a few tokens cost a narrow tile. The K
//                        splits of a tile are one thread-block cluster and are summed through distributed shared memory.
//   product_pair_kernel  CTA pairs (cta_group::2) of 256 x 256 tiles for products with many of them.
// Measured: nvfp4 1x28672x4096 13.6 us (4.85 TB/s: the weights' bytes and 3 us of launch, first loads and epilogue bound
// it), mxfp4 128x4096x14336 12.7 us; 8192x28672x4096 nvfp4 383-408 us from GPU to GPU (4.7-5.0 PFLOP/s), mxfp4 366-376,
// mxfp8 690 (2.8), in launches with pauses between them: back to back for seconds, under the power cap, nvfp4 takes 461.
// With its loads, scales or stores left out the last shape's nvfp4 time falls by some 100, 55 and 45 us: the MMAs alone take
// 244 us, and shared memory's bandwidth, which they share with the copies in and out, is what is between.
// Every wait on an mbarrier is bounded as in b2g_gemm.cu (1 s; less where a plan of single CTAs sets it): on expiry the
// status word gets a code, the CTA's other roles stop, its copies and MMAs in flight land (waits of 50 ms each at most; a
// pair whose issuer gave up relies on its second of waiting for copies that the producers had sent before) and it returns
// without storing. The allocation of tensor memory and the cluster barriers have no limit of their own: the
// first ends because whoever holds columns runs to its end (launch_dependents), the second because every thread of every
// CTA reaches them after bounded waits.

#include <cuda.h>

#include <cstring>
#include <mutex>
#include <new>

#include "micro_common.cuh"
#include "micro_ptx.cuh"

namespace b2g {
namespace micro {

constexpr uint32_t kCtl = 1024;                       // barriers and flags in front of the ring
constexpr int kMaxStages = 16;
constexpr uint64_t kWaitNs = 1000000000ull;           // 1 s per wait unless the plan sets less: far above any legal stall
constexpr uint64_t kDrainNs = 50000000ull;            // 50 ms to drain in-flight work after an abort
constexpr uint32_t kMaxSmem = 232448;                 // sm_100 opt-in maximum dynamic shared memory per block
constexpr int kStepsPerStage = 4;                     // MMAs of 32 bytes of K in a 128-byte stage

constexpr uint32_t O_FULL = 0, O_EMPTY = 128, O_TFULL = 256, O_TEMPTY = 264, O_DRAIN = 272, O_TMEM = 280, O_ABORT = 284;

// status codes: b2g_status_string names them
constexpr int kProducerTimeout = 0x101, kMmaTimeout = 0x102, kEpilogueTimeout = 0x103;

// Scale tiles (4 blocks a row) of a stage's K, and tensor-memory columns and bytes of one 128-row tile's.
constexpr int tiles_of(int kind) { return kind == FMT_MXFP8 ? 1 : kind == FMT_MXFP4 ? 2 : 4; }
// K columns of a stage and of one MMA
constexpr int stage_k(int kind) { return kind == FMT_MXFP8 ? 128 : 256; }
constexpr int step_k(int kind) { return stage_k(kind) / kStepsPerStage; }
// K step `s` of a stage: its scales' tile, and the byte in the tile's cells where they start
constexpr int step_tile(int kind, int s) { return kind == FMT_MXFP8 ? 0 : kind == FMT_MXFP4 ? s / 2 : s; }
constexpr uint32_t step_id(int kind, int s) { return kind == FMT_MXFP8 ? s : kind == FMT_MXFP4 ? (s & 1) * 2 : 0; }

// P: the operand on the MMA's row side (rows_p), Q: the one on its column side.
struct Params {
  int32_t rows_p, rows_q, K, num_kb;
  int32_t tile_q, q_tiles;           // columns of a tile; 128-row scale tiles they span
  int32_t stages, split;
  int32_t tiles_p, tiles_q, units, group;
  uint32_t q_bytes, stage_bytes;     // Q's codes of a stage; its place in the ring, whole KB
  uint32_t tx_bytes;                 // what its copies bring: codes and scales of both operands
  uint32_t acc_cols, tmem_cols;
  void* out;
  int64_t ldc;
  int32_t out_bf16, vec;             // vec: C's rows can be stored in 16-byte pieces
  const float *scale_a, *scale_b;    // NVFP4 tensor scales
  int* status;
  uint64_t wait_ns;
};

// The slow path suspends in slices of at most a quarter of the limit and at most 1 ms, so the limit holds to within one.
__device__ __forceinline__ uint32_t wait_slice(uint64_t limit_ns) {
  return static_cast<uint32_t>(limit_ns / 4 < 1000000ull ? limit_ns / 4 : 1000000ull);
}

__device__ __noinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, int* status,
                                        uint64_t limit_ns, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t slice = wait_slice(limit_ns);
  const uint64_t t0 = global_timer_ns();
  for (;;) {
    if (mbar_try_wait_hint(bar, parity, slice)) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *abort_flag = 1u;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}

// The same for a converged warp, which goes on with one answer: the votes make it, and with it every loop counter and
// descriptor of the warp's loop, uniform in the compiler's eyes. Operands of tcgen05 instructions come from uniform
// registers; from per-thread ones each costs a move of tens of cycles, and the issue, not the tensor core, sets the
// pace.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, int* status,
                                          uint64_t limit_ns, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint32_t slice = wait_slice(limit_ns);
  const uint64_t t0 = global_timer_ns();
  for (;;) {
    if (__all_sync(0xffffffffu, mbar_try_wait_hint(bar, parity, slice))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0u)) return false;
    if (__any_sync(0xffffffffu, global_timer_ns() - t0 > limit_ns)) {
      *abort_flag = 1u;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}

// A value that every lane has, in a uniform register.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

__device__ __noinline__ void drain_phase(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (global_timer_ns() - t0 > limit_ns) return;
  }
}

__device__ __forceinline__ uint32_t cvt2(float a, float b, int bf16) {
  return bf16 ? pack_pair(a, b, static_cast<__nv_bfloat16*>(nullptr)) : pack_pair(a, b, static_cast<__half*>(nullptr));
}

// Both tensor scales as two factors for the accumulators. One large and one small scale are multiplied beforehand; two
// of one kind are applied one after the other, since their product may leave fp32's range where a result does not (and
// a zero times an infinity is none).
__device__ __forceinline__ float2 output_scale(const Params& p) {
  if (!p.scale_a) return make_float2(1.f, 1.f);
  const float a = *p.scale_a, b = *p.scale_b;
  return (a < 1.f) == (b < 1.f) ? make_float2(a, b) : make_float2(a * b, 1.f);
}

// Two accumulators as two values of C.
__device__ __forceinline__ uint32_t result2(float a, float b, float2 scale, int bf16) {
  return cvt2(a * scale.x * scale.y, b * scale.x * scale.y, bf16);
}

// Scales of stage columns in tensor memory: P's tiles first (4 columns each), then Q's, K tile by K tile.
template <int KIND>
__device__ __forceinline__ uint32_t scale_cols(int q_tiles) {
  return tiles_of(KIND) * 4u * (1u + static_cast<uint32_t>(q_tiles));
}

// Four consecutive values of a row of C, `n` of which exist; `vec`: C's rows are 16-byte aligned.
__device__ __forceinline__ void store_four(uint16_t* o, uint2 w, bool vec, int n) {
  if (vec && n >= 4) {
    *reinterpret_cast<uint2*>(o) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) o[k] = static_cast<uint16_t>((k < 2 ? w.x : w.y) >> (16 * (k & 1)));
  }
}

// Issue one stage: its scales into tensor memory, then up to four MMAs (fewer where K ends inside the stage: codes
// past K are zero but the scales there may be any bytes). `sp`, `sq`, `cp`, `cq`: shared addresses of P's and Q's
// codes and of their scales.
template <int KIND, int PAIR>
__device__ __forceinline__ void issue_stage(uint32_t d, uint64_t p_desc, uint64_t q_desc, uint32_t cp, uint32_t cq,
                                            uint32_t tmem_scales, int q_tiles, const uint32_t (&idesc)[kStepsPerStage],
                                            int steps, uint32_t first) {
  constexpr int T = tiles_of(KIND);
  const uint32_t tq = tmem_scales + 4 * T;
  const uint32_t pl = static_cast<uint32_t>(p_desc), ql = static_cast<uint32_t>(q_desc);
#pragma unroll
  for (int k = 0; k < T; ++k) {
    scales_to_tmem_w<PAIR>(tmem_scales + 4 * k, cp + k * 512);
    scales_to_tmem_w<PAIR>(tq + 4 * q_tiles * k, cq + k * 512);
    if (q_tiles == 2) scales_to_tmem_w<PAIR>(tq + 8 * k + 4, cq + (T + k) * 512);
  }
#pragma unroll
  for (int s = 0; s < kStepsPerStage; ++s) {
    if (s < steps)
      umma_scaled_w<KIND, PAIR>(d, pl + s * 2, ql + s * 2, static_cast<uint32_t>(p_desc >> 32), idesc[s],
                                tmem_scales + 4 * step_tile(KIND, s), tq + 4 * q_tiles * step_tile(KIND, s),
                                s == 0 ? first : 1u);
  }
}

template <int KIND>
__global__ void __launch_bounds__(192, 1)
    product_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap map_p,
                   const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_sp,
                   const __grid_constant__ CUtensorMap map_sq) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr uint32_t kPBytes = 128 * 128, kTileBytes = 512u * tiles_of(KIND);
  const uint32_t ctl = smem_addr(smem_raw);
  const uint32_t ring = (ctl + kCtl + 1023u) & ~1023u;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_raw + O_ABORT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = static_cast<int>(blockIdx.x);
  const int tile = unit / p.split, split = unit - tile * p.split;
  const int tp = tile / p.tiles_q, tq = tile - tp * p.tiles_q;
  const int kb0 = static_cast<int>(static_cast<int64_t>(split) * p.num_kb / p.split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(split + 1) * p.num_kb / p.split);

  // Stage `s` of the ring from K block `kb`, by one thread.
  auto load_stage = [&](int s, int kb) {
    const uint32_t full = ctl + O_FULL + 8 * s, base = ring + s * p.stage_bytes;
    mbar_arrive_expect_tx(full, p.tx_bytes);
    tma_load_2d(base, &map_p, full, kb * 128, tp * 128);
    tma_load_2d(base + kPBytes, &map_q, full, kb * 128, tq * p.tile_q);
    tma_load_3d(base + kPBytes + p.q_bytes, &map_sp, full, 0, kb * tiles_of(KIND), tp);
    tma_load_3d(base + kPBytes + p.q_bytes + kTileBytes, &map_sq, full, 0, kb * tiles_of(KIND), tq * p.tile_q / 128);
  };

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_p);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_sp);
    tma_prefetch_desc(&map_sq);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(ctl + O_FULL + 8 * s, 1);
      mbar_init(ctl + O_EMPTY + 8 * s, 1);
    }
    mbar_init(ctl + O_TFULL, 1);
    mbar_init(ctl + O_DRAIN, 1);
    *abort_flag = 0u;
    fence_mbar_init();
    // The first stage goes out while warp 1 allocates tensor memory (one stage: more would hold up the block's
    // barrier).
    asm volatile("griddepcontrol.wait;" ::: "memory");
    load_stage(0, kb0);  // every split has a K block
  }
  if (warp == 1) {
    tmem_alloc(ctl + O_TMEM, p.tmem_cols);
    tmem_relinquish();
    launch_dependents();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + O_TMEM);

  int issued = 1;  // by thread 0: stages whose copies went out
  if (warp == 0) {
    if (lane == 0) {  // TMA producer; the first stage is under way
      int s = 1;
      uint32_t ph = 0;
      for (int kb = kb0 + 1; kb < kb1; ++kb) {
        const uint32_t empty = ctl + O_EMPTY + 8 * s;
        if (!mbar_try_wait(empty, ph ^ 1u) && !wait_phase(empty, ph ^ 1u, abort_flag, p.status, p.wait_ns, kProducerTimeout))
          break;
        load_stage(s, kb);
        ++issued;
        if (++s == p.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {  // MMA issuer: the warp waits together, lane 0 issues
    uint32_t idesc[kStepsPerStage];
#pragma unroll
    for (int i = 0; i < kStepsPerStage; ++i) idesc[i] = idesc_scaled(KIND, step_id(KIND, i), 128, p.tile_q);
    const uint64_t pd = sdesc_sw128(ring, 16u, 1024u), qd = sdesc_sw128(ring + kPBytes, 16u, 1024u);
    const uint32_t cols = scale_cols<KIND>(p.q_tiles), utmem = uniform(tmem);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const uint32_t full = ctl + O_FULL + 8 * s;
      if (!warp_wait(full, ph, abort_flag, p.status, p.wait_ns, kMmaTimeout)) {
        ok = false;
        break;
      }
      const uint32_t base = ring + s * p.stage_bytes, off = s * (p.stage_bytes >> 4);
      const int left = p.K - kb * stage_k(KIND);
      const int steps = left >= stage_k(KIND) ? kStepsPerStage : (left + step_k(KIND) - 1) / step_k(KIND);
      issue_stage<KIND, 0>(utmem, pd + off, qd + off, base + kPBytes + p.q_bytes, base + kPBytes + p.q_bytes + kTileBytes,
                           utmem + p.acc_cols + s * cols, p.q_tiles, idesc, steps, kb == kb0 ? 0u : 1u);
      umma_commit_w(ctl + O_EMPTY + 8 * s);
      if (++s == p.stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    if (ok) umma_commit_w(ctl + O_TFULL);
    umma_commit_w(ctl + O_DRAIN);
    drain_phase(ctl + O_DRAIN, 0, ok ? kWaitNs : kDrainNs);
  } else {
    // Epilogue, part one: this split's fp32 tile into shared memory as [column j][row i] (128 + 4 floats a column: 32
    // lanes store 32 consecutive words). The ring is free: every MMA has completed.
    const int q = warp & 3;
    if (wait_phase(ctl + O_TFULL, 0u, abort_flag, p.status, p.wait_ns, kEpilogueTimeout)) {
      tc_fence_after();
      const int i = q * 32 + lane;
      for (int c = 0; c < p.tile_q; c += 32) {
        const int n = min(32, p.tile_q - c);
        uint32_t v[32];
        const uint32_t at = tmem + c + (static_cast<uint32_t>(q * 32) << 16);
        if (n == 32) tmem_ld_32cols(at, v);
        else tmem_ld_16cols(at, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < n) st_shared_u32(ring + ((c + j) * 132 + i) * 4u, v[j]);
      }
    }
  }
  // Part two: CTA r of the cluster adds its share of the tile over the cluster's CTAs in split order, scales, converts
  // and stores, a lane four consecutive values (a warp's loads of other CTAs' memory are whole lines that way). Every
  // thread of every CTA reaches both barriers. A CTA that gave up stores nothing.
  __syncwarp();
  if (p.split > 1) cluster_sync();
  else __syncthreads();
  const bool gave_up = *abort_flag != 0u;
  if (!gave_up) {
    const float2 alpha = output_scale(p);
    const int cols = min(p.tile_q, p.rows_q - tq * p.tile_q);  // columns of the tile inside C^T
    const int groups = cols * 32;  // of four values
    const int g1 = groups * (split + 1) / p.split;
    uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(tq) * p.tile_q * p.ldc + static_cast<int64_t>(tp) * 128;
    const int rows = p.rows_p - tp * 128;  // the tile's rows inside C^T
    for (int g0 = groups * split / p.split + static_cast<int>(threadIdx.x); g0 < g1; g0 += 2 * 192) {  // two at a time
      float4 v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < p.split; ++s) {
        float4 x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int g = min(g0 + u * 192, g1 - 1);
          const uint32_t off = ring + ((g >> 5) * 132 + (g & 31) * 4) * 4u;
          x[u] = ld_cluster_v4(p.split > 1 ? map_to_rank(off, s) : off);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          v[u].x += x[u].x;
          v[u].y += x[u].y;
          v[u].z += x[u].z;
          v[u].w += x[u].w;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int g = g0 + u * 192, j = g >> 5, i = (g & 31) * 4;
        if (g >= g1 || i >= rows) continue;
        const uint2 w = make_uint2(result2(v[u].x, v[u].y, alpha, p.out_bf16), result2(v[u].z, v[u].w, alpha, p.out_bf16));
        store_four(out + j * p.ldc + i, w, p.vec, rows - i);
      }
    }
  }
  __syncwarp();
  if (p.split > 1) cluster_sync();  // a CTA's shared memory stays until its peers have read it
  else __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
  if (gave_up && threadIdx.x == 0) {
    // Shared memory is released when this thread ends: whichever role gave up, every copy that went out lands first. The
    // last one filled stage (issued - 1) mod stages, in lap (issued - 1) / stages.
    for (int i = issued - 1; i >= 0 && i >= issued - p.stages; --i)
      drain_phase(ctl + O_FULL + 8 * (i % p.stages), static_cast<uint32_t>(i / p.stages) & 1u, kDrainNs);
  }
}

// ---------------------------------------------------------------- CTA pairs
constexpr int kPairEpilogueWarps = 8;
constexpr uint32_t kPairStaging = kPairEpilogueWarps * 4096u;
constexpr int kPartRow = 256 + 4;  // floats a row of a split's part in shared memory

// Tile `t` of the pairs' walk: bands of `group` tile rows, inside a band down the rows first, so that the tiles that
// run at one time share operands in L2.
__device__ __forceinline__ void pair_tile(const Params& p, int t, int& tp, int& tq) {
  const int band = p.group * p.tiles_q;
  const int g = t / band, r = t - g * band;
  const int h = min(p.group, p.tiles_p - g * p.group);
  tq = r / h;
  tp = g * p.group + (r - tq * h);
}

// 256 x 256 tiles, a persistent CTA pair on each (or, with K split, the pairs of a cluster on one tile, a K range
// each): every CTA loads its 128 rows of P, half of Q's 256 and the scales of its P rows and of all of Q (both tensor
// memories hold Q's scales), the leader issues MMAs of M = 256, and each CTA ends with a 128 x 256 accumulator. 256
// accumulator columns and the stages' scales fill tensor memory, so there is one accumulator: the epilogue's eight
// warps read it into registers and free it before they convert the second half and store, while the next tile's MMAs
// run.
template <int KIND>
__global__ void __launch_bounds__((2 + kPairEpilogueWarps) * 32, 1)
    product_pair_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap map_p,
                        const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_sp,
                        const __grid_constant__ CUtensorMap map_sq, const __grid_constant__ CUtensorMap map_c) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr uint32_t kPBytes = 128 * 128, kTileBytes = 512u * tiles_of(KIND);
  const uint32_t ctl = smem_addr(smem_raw);
  const uint32_t ring = (ctl + kCtl + 1023u) & ~1023u;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_raw + O_ABORT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_ctarank());
  const int rank = cta & 1, split = cta >> 1;  // within the pair; the pair's K split
  const uint32_t lead = static_cast<uint32_t>(cta & ~1);
  const bool leader = rank == 0;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(num_clusters_x());
  const int kb0 = static_cast<int>(static_cast<int64_t>(split) * p.num_kb / p.split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(split + 1) * p.num_kb / p.split);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_p);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_sp);
    tma_prefetch_desc(&map_sq);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(ctl + O_FULL + 8 * s, 1);
      mbar_init(ctl + O_EMPTY + 8 * s, 1);
    }
    mbar_init(ctl + O_TFULL, 1);
    mbar_init(ctl + O_TEMPTY, 2 * kPairEpilogueWarps);  // one arrival per epilogue warp of both CTAs, at the leader's
    mbar_init(ctl + O_DRAIN, 1);
    *abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(ctl + O_TMEM, p.tmem_cols);
    tmem_relinquish_pair();
    launch_dependents();
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist before any signal crosses
  tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + O_TMEM);

  if (warp == 0) {
    if (lane == 0) {  // TMA producer: each CTA's copies count on the leader's barriers
      const uint32_t full0 = map_to_rank(ctl + O_FULL, lead);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; ok && t < p.units; t += step) {
        int tp, tq;
        pair_tile(p, t, tp, tq);
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t empty = ctl + O_EMPTY + 8 * s, full = full0 + 8 * s;
          if (!mbar_try_wait(empty, ph ^ 1u) &&
              !wait_phase(empty, ph ^ 1u, abort_flag, p.status, p.wait_ns, kProducerTimeout)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(ctl + O_FULL + 8 * s, p.tx_bytes);
          const uint32_t base = ring + s * p.stage_bytes;
          tma_load_2d_pair(base, &map_p, full, kb * 128, tp * 256 + rank * 128);
          tma_load_2d_pair(base + kPBytes, &map_q, full, kb * 128, tq * 256 + rank * 128);
          tma_load_3d_pair(base + kPBytes + p.q_bytes, &map_sp, full, 0, kb * tiles_of(KIND), tp * 2 + rank);
          tma_load_3d_pair(base + kPBytes + p.q_bytes + kTileBytes, &map_sq, full, 0, kb * tiles_of(KIND), tq * 2);
          ++issued;
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok && leader) {  // the leader's barriers count the pair's copies: let those already issued land
        for (int i = min(issued, p.stages); i > 0; --i) {
          if (--s < 0) {
            s = p.stages - 1;
            ph ^= 1u;
          }
          drain_phase(ctl + O_FULL + 8 * s, ph, kDrainNs);
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {  // MMA issuer for both CTAs
      uint32_t idesc[kStepsPerStage];
#pragma unroll
      for (int i = 0; i < kStepsPerStage; ++i) idesc[i] = idesc_scaled(KIND, step_id(KIND, i), 256, 256);
      const uint64_t pd = sdesc_sw128(ring, 16u, 1024u), qd = sdesc_sw128(ring + kPBytes, 16u, 1024u);
      constexpr uint32_t cols = tiles_of(KIND) * 12u;  // a stage's scales: one tile row of P, two of Q
      const uint32_t empty0 = map_to_rank(ctl + O_EMPTY, lead), empty1 = map_to_rank(ctl + O_EMPTY, lead + 1);
      const uint32_t utmem = uniform(tmem);
      const uint32_t tfull0 = map_to_rank(ctl + O_TFULL, lead), tfull1 = map_to_rank(ctl + O_TFULL, lead + 1);
      const int last = p.K - (p.num_kb - 1) * stage_k(KIND);
      const int last_steps = (last + step_k(KIND) - 1) / step_k(KIND);
      int s = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = first; ok && t < p.units; t += step) {
        if (!warp_wait(ctl + O_TEMPTY, acc_ph ^ 1u, abort_flag, p.status, p.wait_ns, kMmaTimeout)) {
          ok = false;
          break;
        }
        acc_ph ^= 1u;
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t full = ctl + O_FULL + 8 * s;
          if (!warp_wait(full, ph, abort_flag, p.status, p.wait_ns, kMmaTimeout)) {
            ok = false;
            break;
          }
          const uint32_t base = ring + s * p.stage_bytes, off = s * (p.stage_bytes >> 4);
          issue_stage<KIND, 1>(utmem, pd + off, qd + off, base + kPBytes + p.q_bytes,
                               base + kPBytes + p.q_bytes + kTileBytes, utmem + p.acc_cols + s * cols, 2, idesc,
                               kb + 1 == p.num_kb ? last_steps : kStepsPerStage, kb == kb0 ? 0u : 1u);
          umma_commit_pair_w(empty0 + 8 * s);
          umma_commit_pair_w(empty1 + 8 * s);
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair_w(tfull0);
        umma_commit_pair_w(tfull1);
      }
      umma_commit_pair_w(map_to_rank(ctl + O_DRAIN, lead));
      drain_phase(ctl + O_DRAIN, 0, ok ? kWaitNs : kDrainNs);
    }
  } else {
    const int e = warp - 2, q = warp & 3, half = e >> 2;  // tensor-memory lane quarter, half of the columns
    const uint32_t tempty = map_to_rank(ctl + O_TEMPTY, lead);
    const uint32_t stg = ring + p.stages * p.stage_bytes + static_cast<uint32_t>(e) * 4096u;
    const float2 alpha = output_scale(p);
    uint16_t* out = static_cast<uint16_t*>(p.out);
    uint32_t ph = 0;
    for (int t = first; t < p.units; t += step) {
      int tp, tq;
      pair_tile(p, t, tp, tq);
      if (!wait_phase(ctl + O_TFULL, ph, abort_flag, p.status, p.wait_ns, kEpilogueTimeout)) break;
      ph ^= 1u;
      tc_fence_after();
      if (p.split > 1) {  // the pair's only tile: this split's part of it stays in shared memory, fp32 (below)
        const uint32_t to = ring + static_cast<uint32_t>((q * 32 + lane) * kPartRow + half * 128) * 4u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld_32cols(tmem + half * 128 + c * 32 + (static_cast<uint32_t>(q * 32) << 16), v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            st_shared_v4(to + (c * 32 + 4 * j) * 4u, make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        break;
      }
      uint32_t w[64];  // the row's 128 columns, rounded
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          tmem_ld_32cols(tmem + half * 128 + h * 64 + c * 32 + (static_cast<uint32_t>(q * 32) << 16), v[c]);
        tmem_ld_wait();
        if (h == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            w[h * 32 + c * 16 + j] =
                result2(__uint_as_float(v[c][2 * j]), __uint_as_float(v[c][2 * j + 1]), alpha, p.out_bf16);
      }
      const int64_t row0 = static_cast<int64_t>(tp) * 256 + rank * 128 + q * 32;
      const int64_t col0 = static_cast<int64_t>(tq) * 256 + half * 128;
      if (p.vec) {
        // 32 rows x 64 columns at a time through the warp's 4 KB of shared memory (16-byte pieces XOR-ed by the row,
        // the 128-byte swizzle) and out by TMA, which writes whole lines and drops what lies outside C
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (lane == 0) tma_store_wait_read();  // the last store has read the buffer
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            st_shared_v4(stg + lane * 128 + ((j ^ (lane & 7)) << 4),
                         make_uint4(w[h * 32 + 4 * j], w[h * 32 + 4 * j + 1], w[h * 32 + 4 * j + 2], w[h * 32 + 4 * j + 3]));
          fence_async_shared();
          __syncwarp();
          if (lane == 0) tma_store_2d(&map_c, stg, static_cast<int32_t>(col0) + h * 64, static_cast<int32_t>(row0));
        }
      } else {  // rows of C that are not 16-byte aligned: through the same buffer, 32 consecutive values an instruction
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            st_shared_v4(stg + lane * 128 + ((j ^ (lane & 7)) << 4),
                         make_uint4(w[h * 32 + 4 * j], w[h * 32 + 4 * j + 1], w[h * 32 + 4 * j + 2], w[h * 32 + 4 * j + 3]));
          __syncwarp();
          const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.rows_p - row0));
          for (int r = 0; r < rows; ++r) {
            uint16_t* o = out + (row0 + r) * p.ldc + col0 + h * 64;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int c = k * 32 + lane;
              if (col0 + h * 64 + c < p.rows_q) o[c] = ld_shared_u16(stg + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) tma_store_wait();
  }
  __syncwarp();
  cluster_sync();  // the pair's MMAs and signals are done in both CTAs; the splits' parts lie in shared memory
  if (p.split > 1) {
    // Each CTA adds its share of the columns of its 128 rows over the splits, in split order, from the CTAs of its
    // rank in every pair; the rows were stored 4 floats apart in banks. Then the cluster's shared memory may go.
    int tp, tq;
    pair_tile(p, first, tp, tq);
    const float2 alpha = output_scale(p);
    const int per0 = 64 * split / p.split, per = 64 * (split + 1) / p.split - per0;  // groups of four columns a row
    const int64_t row0 = static_cast<int64_t>(tp) * 256 + rank * 128, col0 = static_cast<int64_t>(tq) * 256 + per0 * 4;
    auto sum = [&](auto splits) {
      constexpr int S = decltype(splits)::value, kThreads = (2 + kPairEpilogueWarps) * 32;
      constexpr int kGroups = 16 / S;  // a thread's sixteen loads in flight: other CTAs' memory is far away
      for (int g0 = static_cast<int>(threadIdx.x); g0 < 128 * per; g0 += kGroups * kThreads) {
        float4 x[kGroups][S];
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
          const int g = g0 + u * kThreads, i = g / per;
          const uint32_t off = ring + static_cast<uint32_t>(i * kPartRow + (per0 + g - i * per) * 4) * 4u;
          if (g < 128 * per) {
#pragma unroll
            for (int k = 0; k < S; ++k) x[u][k] = ld_cluster_v4(map_to_rank(off, 2 * k + rank));
          }
        }
#pragma unroll
        for (int u = 0; u < kGroups; ++u) {
          const int g = g0 + u * kThreads, i = g / per, j = (g - i * per) * 4;
          if (g >= 128 * per || row0 + i >= p.rows_p || col0 + j >= p.rows_q) continue;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < S; ++k) {
            v.x += x[u][k].x;
            v.y += x[u][k].y;
            v.z += x[u][k].z;
            v.w += x[u][k].w;
          }
          uint16_t* o = static_cast<uint16_t*>(p.out) + (row0 + i) * p.ldc + col0 + j;
          const uint2 w = make_uint2(result2(v.x, v.y, alpha, p.out_bf16), result2(v.z, v.w, alpha, p.out_bf16));
          store_four(o, w, p.vec, static_cast<int>(min(static_cast<int64_t>(4), p.rows_q - col0 - j)));
        }
      }
    };
    if (p.split == 2) sum(std::integral_constant<int, 2>{});
    else sum(std::integral_constant<int, 3>{});
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) tmem_dealloc_pair(tmem, p.tmem_cols);
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static std::once_flag once;
  static EncodeFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(f);
    else
      cudaGetLastError();
  });
  return fn;
}

// Codes as rows of bytes: boxes of 128 bytes x `box_rows` rows, 128-byte swizzle. What lies past a row's last code
// byte reads as zero.
int32_t encode_codes(CUtensorMap* map, const b2g_micro_tensor* t, int box_rows) {
  const EncodeFn fn = encode_fn();
  if (!fn) return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int64_t bytes = t->format == FMT_MXFP8 ? t->cols : (t->cols + 1) / 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(t->rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(t->pitch)};
  const cuuint32_t box[2] = {128u, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t->codes, dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return B2G_OK;
  return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled (codes): error " + std::to_string(static_cast<int>(r)));
}

// Scales as [row tile][K tile][512 bytes]: boxes of `ktiles` K tiles x `row_tiles` row tiles. Tiles that do not exist
// read as zero.
int32_t encode_scales(CUtensorMap* map, const b2g_micro_tensor* t, int ktiles, int row_tiles) {
  const EncodeFn fn = encode_fn();
  if (!fn) return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int64_t kt = ceil_div(t->cols, 4 * block_of(t->format));
  const cuuint64_t dims[3] = {128u, static_cast<cuuint64_t>(kt), static_cast<cuuint64_t>(ceil_div(t->rows, 128))};
  const cuuint64_t strides[2] = {512u, static_cast<cuuint64_t>(kt * 512)};
  const cuuint32_t box[3] = {128u, static_cast<cuuint32_t>(ktiles), static_cast<cuuint32_t>(row_tiles)};
  const cuuint32_t elem[3] = {1u, 1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, t->scales, dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return B2G_OK;
  return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled (scales): error " + std::to_string(static_cast<int>(r)));
}

// C in boxes of 32 rows x 64 columns for the pairs' stores (16-byte aligned rows only).
int32_t encode_out(CUtensorMap* map, const Params& p) {
  const EncodeFn fn = encode_fn();
  if (!fn) return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.rows_q), static_cast<cuuint64_t>(p.rows_p)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ldc) * 2};
  const cuuint32_t box[2] = {64u, 32u};
  const cuuint32_t elem[2] = {1u, 1u};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.out, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return B2G_OK;
  return record_error(B2G_ERR_CUDA, "cuTensorMapEncodeTiled (C): error " + std::to_string(static_cast<int>(r)));
}

// Function attributes, once per device.
int32_t init_device(int dev) {
  static std::mutex mu;
  static bool done[64];
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && dev < 64 && done[dev]) return B2G_OK;
  const void* fns[] = {reinterpret_cast<const void*>(product_kernel<FMT_MXFP8>),
                       reinterpret_cast<const void*>(product_kernel<FMT_MXFP4>),
                       reinterpret_cast<const void*>(product_kernel<FMT_NVFP4>),
                       reinterpret_cast<const void*>(product_pair_kernel<FMT_MXFP8>),
                       reinterpret_cast<const void*>(product_pair_kernel<FMT_MXFP4>),
                       reinterpret_cast<const void*>(product_pair_kernel<FMT_NVFP4>)};
  for (const void* f : fns) {
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return record_error(B2G_ERR_CUDA, std::string("kernel attributes: ") + cudaGetErrorString(e));
    }
  }
  if (dev >= 0 && dev < 64) done[dev] = true;
  return B2G_OK;
}

// Clusters of 1..8 CTAs with the whole shared memory of an SM each that the measured B200 holds at once (a cluster lives
// inside a GPC): a launch of more runs in waves, with the same results.
constexpr int kClusters[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};

constexpr int kPairs = 74;  // CTA pairs resident at once

// K splits of a single-CTA product of `tiles` tiles: one cluster a tile, as many splits as keep every cluster resident
// at once and leave each split two stages.
int splits(int64_t tiles, int num_kb) {
  int split = 1;
  for (int s = 2; s <= 8; ++s)
    if (tiles <= kClusters[s] && num_kb >= 2 * s) split = s;
  return split;
}

// Pairs, unless a side fits one 128-row tile, or there are so few 128 x 128 tiles that single CTAs split K over the
// GPU and K is long enough to gain by it. Measured, pairs against single CTAs (us): nvfp4 512x4096x4096 (no split)
// 10.9, 13.6; 256x28672x4096 22.1, 30.3; 256x4096x4096 (two splits of 16 stages) 10.6, 9.5; 256x4096x14336 17.3, 15.4;
// 1024^3 (two splits of 4 stages) 6.2, 7.6; mxfp8 512x2048x2048 (of 16) 9.9, 9.2; 1024^3 (of 8) 7.2, 8.0.
bool use_pairs(int64_t M, int64_t N, int num_kb) {
  if (M <= 128 || N <= 128) return false;
  return num_kb <= 8 || splits(ceil_div(M, 128) * ceil_div(N, 128), num_kb) == 1;
}

// K splits of a product of `tiles` pairs' tiles: the pairs of one cluster, while every cluster is resident at once.
// Adding the parts through distributed shared memory takes 4-5 us, the time of some 18 stages, so that many have to be
// saved (four splits never do: so few tiles have single CTAs split K): 512x4096x14336 (two splits) nvfp4 23.9 -> 20.0
// us, mxfp8 40.0 -> 29.7; at K = 4096 nvfp4 10.9 -> 12.9.
int pair_splits(int64_t tiles, int num_kb) {
  int split = 1;
  for (int s = 2; s <= 3; ++s)
    if (tiles <= kClusters[2 * s] && num_kb * (s - 1) >= 18 * s) split = s;
  return split;
}

struct Plan {
  Params p;
  CUtensorMap map_p, map_q, map_sp, map_sq, map_c;
  int kind, device, grid;
  bool pair;
  uint32_t smem;
  bool empty;    // no output element
  bool zero;     // K = 0: C is zero
  int64_t M, N;
};

uint32_t pow2_cols(uint32_t x) {
  uint32_t c = 32;
  while (c < x) c <<= 1;
  return c;
}

int32_t plan_init(Plan& pl, const b2g_micro_tensor* a, const b2g_micro_tensor* b, void* C, int64_t ldc, int32_t dtype,
                  int32_t* status) {
  if (const int32_t rc = check_tensor(a, "a")) return rc;
  if (const int32_t rc = check_tensor(b, "b")) return rc;
  if (a->format != b->format) return record_error(B2G_ERR_UNSUPPORTED, "format_mismatch: a and b need one format");
  if (a->cols != b->cols) return record_error(B2G_ERR_INVALID_ARG, "a and b differ in columns (the dimension summed over)");
  if (dtype != B2G_VALUE_F16 && dtype != B2G_VALUE_BF16)
    return record_error(B2G_ERR_INVALID_ARG, "dtype must be B2G_VALUE_F16 or B2G_VALUE_BF16");
  pl.M = a->rows;
  pl.N = b->rows;
  pl.kind = a->format;
  pl.empty = pl.M == 0 || pl.N == 0;
  if (pl.M > INT32_MAX - 512 || pl.N > INT32_MAX - 512)
    return record_error(B2G_ERR_UNSUPPORTED, "dimension_too_large: a product needs M and N < 2^31 - 512");
  pl.zero = a->cols == 0;
  if (pl.empty) return B2G_OK;
  if (!C || ldc < pl.N) return record_error(B2G_ERR_INVALID_ARG, "null C or ldc below N");
  // Encoding tensor maps needs the device's context bound to this thread, which a thread that has not used the runtime
  // yet (autograd's own, for one) does not have; naming its current device binds it.
  if (cudaGetDevice(&pl.device) != cudaSuccess || cudaSetDevice(pl.device) != cudaSuccess) {
    cudaGetLastError();
    return record_error(B2G_ERR_CUDA, "no CUDA device");
  }
  Params& p = pl.p;
  std::memset(&p, 0, sizeof p);
  p.out = C;
  p.ldc = ldc;
  if (pl.zero) return B2G_OK;
  if (const int32_t rc = init_device(pl.device)) return rc;
  p.out_bf16 = dtype == B2G_VALUE_BF16;
  p.vec = aligned16(C) && ldc % 8 == 0;
  p.status = status;
  p.wait_ns = kWaitNs;
  if (pl.kind == FMT_NVFP4) {
    p.scale_a = a->scale;
    p.scale_b = b->scale;
  }
  p.K = static_cast<int32_t>(a->cols);
  p.num_kb = static_cast<int32_t>(ceil_div(a->cols, stage_k(pl.kind)));
  const int T = tiles_of(pl.kind);
  pl.pair = use_pairs(pl.M, pl.N, p.num_kb);
  if (pl.pair) {  // rows run over A, columns over B: C's rows are stored as they lie
    p.rows_p = static_cast<int32_t>(pl.M);
    p.rows_q = static_cast<int32_t>(pl.N);
    p.tile_q = 256;
    p.q_tiles = 2;
    p.tiles_p = static_cast<int32_t>(ceil_div(pl.M, 256));
    p.tiles_q = static_cast<int32_t>(ceil_div(pl.N, 256));
    const int64_t tiles = static_cast<int64_t>(p.tiles_p) * p.tiles_q;
    if (tiles > kMaxGrid / 2) return too_large("product");
    p.units = static_cast<int32_t>(tiles);
    p.group = 16;
    p.split = pair_splits(tiles, p.num_kb);
    pl.grid = 2 * p.split * (tiles < kPairs ? static_cast<int>(tiles) : kPairs);
    p.q_bytes = 128u * 128u;
    const uint32_t cta_bytes = 2u * 128u * 128u + 512u * T * 3;
    p.tx_bytes = 2u * cta_bytes;
    p.stage_bytes = (cta_bytes + 1023u) & ~1023u;
    p.acc_cols = 256;
    p.tmem_cols = 512;
    const uint32_t cols = T * 4u * 3u;
    uint32_t stages = (kMaxSmem - 2048u - kPairStaging) / p.stage_bytes;
    if (stages > 256u / cols) stages = 256u / cols;
    p.stages = static_cast<int32_t>(stages);
    pl.smem = kMaxSmem;
    std::memset(&pl.map_c, 0, sizeof pl.map_c);
    if (p.vec)
      if (const int32_t rc = encode_out(&pl.map_c, p)) return rc;
    if (const int32_t rc = encode_codes(&pl.map_p, a, 128)) return rc;
    if (const int32_t rc = encode_codes(&pl.map_q, b, 128)) return rc;
    if (const int32_t rc = encode_scales(&pl.map_sp, a, T, 1)) return rc;
    return encode_scales(&pl.map_sq, b, T, 2);
  }
  // rows run over B, columns over A
  p.rows_p = static_cast<int32_t>(pl.N);
  p.rows_q = static_cast<int32_t>(pl.M);
  p.tile_q = pl.M <= 16 ? 16 : pl.M <= 32 ? 32 : pl.M <= 64 ? 64 : 128;
  p.q_tiles = 1;
  p.tiles_p = static_cast<int32_t>(ceil_div(p.rows_p, 128));
  p.tiles_q = static_cast<int32_t>(ceil_div(p.rows_q, p.tile_q));
  const int64_t tiles = static_cast<int64_t>(p.tiles_p) * p.tiles_q;
  p.split = splits(tiles, p.num_kb);
  if (tiles * p.split > kMaxGrid) return too_large("product");
  p.units = static_cast<int32_t>(tiles * p.split);
  pl.grid = p.units;
  p.q_bytes = static_cast<uint32_t>(p.tile_q) * 128u;
  p.tx_bytes = 128u * 128u + p.q_bytes + 512u * T * (1 + p.q_tiles);
  p.stage_bytes = (p.tx_bytes + 1023u) & ~1023u;
  p.acc_cols = pow2_cols(p.tile_q);
  // Shared memory: clusters take a whole SM's each, so that no CTA of another launch can hold tensor memory there
  // while this cluster's CTAs wait for one another; single CTAs take at most half, two to an SM, and at most half of
  // the tensor memory.
  const uint32_t room = p.split > 1 ? kMaxSmem : 113u * 1024u;
  const uint32_t cols = tiles_of(pl.kind) * 4u * (1u + p.q_tiles);
  uint32_t stages = (room - 2048u) / p.stage_bytes;
  const uint32_t most_cols = p.split > 1 ? 512u : 256u;
  if (stages > (most_cols - p.acc_cols) / cols) stages = (most_cols - p.acc_cols) / cols;
  if (stages > static_cast<uint32_t>(kMaxStages)) stages = kMaxStages;
  p.stages = static_cast<int32_t>(stages);
  p.tmem_cols = pow2_cols(p.acc_cols + stages * cols);
  uint32_t ring = stages * p.stage_bytes;
  const uint32_t tile_bytes = static_cast<uint32_t>(p.tile_q) * 132u * 4u;
  if (ring < tile_bytes) ring = tile_bytes;
  pl.smem = p.split > 1 ? kMaxSmem : 2048u + ring;
  if (p.split == 1 && pl.smem < 78u * 1024u) pl.smem = 78u * 1024u;  // never three to an SM: tensor memory holds two
  if (const int32_t rc = encode_codes(&pl.map_p, b, 128)) return rc;
  if (const int32_t rc = encode_codes(&pl.map_q, a, p.tile_q)) return rc;
  if (const int32_t rc = encode_scales(&pl.map_sp, b, T, 1)) return rc;
  return encode_scales(&pl.map_sq, a, T, p.q_tiles);
}

int32_t plan_launch(const Plan& pl, cudaStream_t st) {
  if (pl.empty) return B2G_OK;
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != pl.device) {
    cudaGetLastError();
    return record_error(B2G_ERR_INVALID_ARG, "plan was made on device " + std::to_string(pl.device) + " but device " +
                                                 std::to_string(cur) + " is current");
  }
  if (pl.zero) {
    const cudaError_t e = cudaMemset2DAsync(pl.p.out, static_cast<size_t>(pl.p.ldc) * 2, 0, static_cast<size_t>(pl.N) * 2,
                                            static_cast<size_t>(pl.M), st);
    if (e == cudaSuccess) return B2G_OK;
    cudaGetLastError();
    return record_error(B2G_ERR_CUDA, std::string("memset: ") + cudaGetErrorString(e));
  }
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  lc.stream = st;
  lc.gridDim = dim3(static_cast<unsigned>(pl.grid), 1, 1);
  lc.blockDim = dim3(pl.pair ? (2 + kPairEpilogueWarps) * 32 : 192, 1, 1);
  lc.dynamicSmemBytes = pl.smem;
  const int cluster = pl.pair ? 2 * pl.p.split : pl.p.split;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    lc.numAttrs = 2;
  }
  cudaError_t e = cudaSuccess;
  by_format(pl.kind, [&](auto f) -> int32_t {
    constexpr int F = decltype(f)::value;
    e = pl.pair ? cudaLaunchKernelEx(&lc, product_pair_kernel<F>, pl.p, pl.map_p, pl.map_q, pl.map_sp, pl.map_sq, pl.map_c)
                : cudaLaunchKernelEx(&lc, product_kernel<F>, pl.p, pl.map_p, pl.map_q, pl.map_sp, pl.map_sq);
    return B2G_OK;
  });
  if (e == cudaSuccess) return B2G_OK;
  cudaGetLastError();
  return record_error(B2G_ERR_CUDA, std::string("product launch: ") + cudaGetErrorString(e));
}

// Where the quantised operands of a product of values lie in its workspace: A's tensor scale, B's, then codes and scales
// of each. Every part is a multiple of 16 bytes.
struct ValuesLayout {
  b2g_micro_tensor a, b;
  size_t bytes;
};

ValuesLayout values_layout(int fmt, int64_t M, int64_t N, int64_t K, uint8_t* base) {
  ValuesLayout l;
  size_t at = 32;
  const auto place = [&](int64_t rows, size_t scale_at) {
    b2g_micro_tensor t = {};
    t.format = fmt;
    t.rows = rows;
    t.cols = K;
    t.pitch = min_pitch(fmt, K);
    t.codes = base + at;
    at += static_cast<size_t>(rows * t.pitch);
    t.scales = base + at;
    at += static_cast<size_t>(ceil_div(rows, 128) * ceil_div(K, 4 * block_of(fmt)) * 512);
    t.scale = fmt == FMT_NVFP4 ? reinterpret_cast<const float*>(base + scale_at) : nullptr;
    return t;
  };
  l.a = place(M, 0);
  l.b = place(N, 16);
  l.bytes = at;
  return l;
}

}  // namespace micro
}  // namespace b2g

using namespace b2g;
using namespace b2g::micro;

struct b2g_micro_plan {
  Plan plan;
};

extern "C" {

int32_t b2g_micro_plan_create(const b2g_micro_tensor* a, const b2g_micro_tensor* b, void* C, int64_t ldc, int32_t dtype,
                              int32_t* status, b2g_micro_plan** out) {
  return guarded([&]() -> int32_t {
    if (!out) return record_error(B2G_ERR_INVALID_ARG, "null plan output");
    *out = nullptr;
    b2g_micro_plan* p = new (std::nothrow) b2g_micro_plan();
    if (!p) return record_error(B2G_ERR_CUDA, "out of host memory");
    const int32_t rc = plan_init(p->plan, a, b, C, ldc, dtype, status);
    if (rc != B2G_OK) {
      delete p;
      return rc;
    }
    *out = p;
    return B2G_OK;
  });
}

int32_t b2g_micro_plan_launch(const b2g_micro_plan* plan, void* stream) {
  return guarded([&]() -> int32_t {
    if (!plan) return record_error(B2G_ERR_INVALID_ARG, "null plan");
    return plan_launch(plan->plan, static_cast<cudaStream_t>(stream));
  });
}

int32_t b2g_micro_plan_wait_limit(b2g_micro_plan* plan, int32_t wait_limit_us) {
  return guarded([&]() -> int32_t {
    if (!plan) return record_error(B2G_ERR_INVALID_ARG, "null plan");
    if (wait_limit_us < 0) return record_error(B2G_ERR_INVALID_ARG, "wait_limit_us must be >= 0");
    Plan& pl = plan->plan;
    if (pl.empty || pl.zero) return B2G_OK;  // nothing waits
    if (wait_limit_us > 0 && (pl.pair || pl.p.split > 1))
      return record_error(B2G_ERR_UNSUPPORTED, "wait_limit_single_cta_only: CTA pairs and the splits of a cluster keep the "
                                               "default wait limit (an early stop cannot wait out other CTAs' copies)");
    pl.p.wait_ns = wait_limit_us > 0 ? static_cast<uint64_t>(wait_limit_us) * 1000ull : kWaitNs;
    return B2G_OK;
  });
}

int32_t b2g_micro_plan_destroy(b2g_micro_plan* plan) {
  delete plan;
  return B2G_OK;
}

int32_t b2g_micro_matmul(const b2g_micro_tensor* a, const b2g_micro_tensor* b, void* C, int64_t ldc, int32_t dtype,
                         int32_t* status, void* stream) {
  return guarded([&]() -> int32_t {
    Plan pl;
    if (const int32_t rc = plan_init(pl, a, b, C, ldc, dtype, status)) return rc;
    return plan_launch(pl, static_cast<cudaStream_t>(stream));
  });
}

int32_t b2g_micro_matmul_values_workspace(int32_t format, int64_t M, int64_t N, int64_t K, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (format < FMT_MXFP8 || format > FMT_NVFP4 || M < 0 || N < 0 || K < 0 || !bytes)
      return record_error(B2G_ERR_INVALID_ARG, "matmul_values_workspace: bad format, dimension or output pointer");
    *bytes = values_layout(format, M, N, K, nullptr).bytes;
    return B2G_OK;
  });
}

int32_t b2g_micro_matmul_values(const b2g_micro_matrix* A, const b2g_micro_matrix* B, int64_t M, int64_t N, int64_t K,
                                int32_t value_dtype, int32_t format, void* C, int64_t ldc, int32_t dtype,
                                void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  return guarded([&]() -> int32_t {
    if (format < FMT_MXFP8 || format > FMT_NVFP4 || M < 0 || N < 0 || K < 0)
      return record_error(B2G_ERR_INVALID_ARG, "matmul_values: bad format or dimension");
    const ValuesLayout l = values_layout(format, M, N, K, static_cast<uint8_t*>(workspace));
    if (!workspace || !aligned16(workspace) || workspace_bytes < l.bytes)
      return record_error(B2G_ERR_WORKSPACE, "matmul_values: workspace missing, misaligned or too small");
    Plan pl;  // checks everything before the first launch
    if (const int32_t rc = plan_init(pl, &l.a, &l.b, C, ldc, dtype, status)) return rc;
    if (!pl.empty && !pl.zero) {
      const b2g_micro_matrix* values[] = {A, B};
      const b2g_micro_tensor* to[] = {&l.a, &l.b};
      for (int i = 0; i < 2; ++i) {
        if (format == FMT_NVFP4)
          if (const int32_t rc = b2g_micro_tensor_scale(values[i], to[i]->rows, K, value_dtype,
                                                        const_cast<float*>(to[i]->scale), stream))
            return rc;
        if (const int32_t rc = b2g_micro_quantize(values[i], value_dtype, to[i], stream)) return rc;
      }
    }
    return plan_launch(pl, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

// micro_ptx.cuh — PTX wrappers the block-scaled products add to b2g_ptx.cuh: block-scaled tcgen05 MMAs, the copy of
// scales from shared to tensor memory, and their descriptors.
#pragma once

#include "b2g_ptx.cuh"

namespace b2g {

// D[tmem] (+)= (A * scale A) * (B * scale B), A and B from shared memory, scales from tensor memory, fp32
// accumulators. KIND 1: 8-bit floats, K = 32, one power-of-two scale per row (kind::mxf8f6f4); 2: e2m1, K = 64, two
// power-of-two scales per row (kind::mxf4); 3: e2m1, K = 64, four e4m3 scales per row (kind::mxf4nvf4). Issued by lane
// 0 of a converged warp. `a`, `b`: the descriptors' low words; `hi`: the high word both share (what varies between
// stages and K steps is the start address, so only one word is computed).
template <int KIND, int PAIR>
__device__ __forceinline__ void umma_scaled_w(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t sa,
                                              uint32_t sb, uint32_t accumulate) {
#define B2G_UMMA_SCALED(GROUP, SPEC)                                                                 \
  asm volatile(                                                                                      \
      "{\n\t.reg .pred p, q;\n\t.reg .u32 l;\n\t.reg .b64 da, db;\n\t"                               \
      "mov.b64 da, {%1, %3};\n\t"                                                                    \
      "mov.b64 db, {%2, %3};\n\t"                                                                    \
      "mov.u32 l, %%laneid;\n\t"                                                                     \
      "setp.eq.u32 q, l, 0;\n\t"                                                                     \
      "setp.ne.b32 p, %7, 0;\n\t"                                                                    \
      "@q tcgen05.mma.cta_group::" GROUP "." SPEC " [%0], da, db, %4, [%5], [%6], p;\n\t}" ::"r"(d), \
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                         \
      : "memory")
  if constexpr (KIND == 1) {
    if constexpr (PAIR) B2G_UMMA_SCALED("2", "kind::mxf8f6f4.block_scale.scale_vec::1X");
    else B2G_UMMA_SCALED("1", "kind::mxf8f6f4.block_scale.scale_vec::1X");
  } else if constexpr (KIND == 2) {
    if constexpr (PAIR) B2G_UMMA_SCALED("2", "kind::mxf4.block_scale.scale_vec::2X");
    else B2G_UMMA_SCALED("1", "kind::mxf4.block_scale.scale_vec::2X");
  } else {
    if constexpr (PAIR) B2G_UMMA_SCALED("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
    else B2G_UMMA_SCALED("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  }
#undef B2G_UMMA_SCALED
}

// A 512-byte scale tile (32 rows of 16 bytes) at shared address `from` into four tensor-memory columns, repeated in
// each quarter of the lanes. The descriptor has no swizzle: 8-row groups of 16 bytes a row, 128 bytes apart.
template <int PAIR>
__device__ __forceinline__ void scales_to_tmem_w(uint32_t tmem, uint32_t from) {
#define B2G_SCALE_COPY(GROUP)                                                           \
  asm volatile(                                                                         \
      "{\n\t.reg .pred q;\n\t.reg .u32 l;\n\t.reg .b64 da;\n\t"                         \
      "mov.b64 da, {%1, %2};\n\t"                                                       \
      "mov.u32 l, %%laneid;\n\t"                                                        \
      "setp.eq.u32 q, l, 0;\n\t"                                                        \
      "@q tcgen05.cp.cta_group::" GROUP ".32x128b.warpx4 [%0], da;\n\t}" ::"r"(tmem),   \
      "r"(from >> 4 | 1u << 16), "r"(8u | 1u << 14)                                     \
      : "memory")
  if constexpr (PAIR) B2G_SCALE_COPY("2");
  else B2G_SCALE_COPY("1");
#undef B2G_SCALE_COPY
}

__device__ __forceinline__ uint16_t ld_shared_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}

// 2-D tile shared -> global; what lies outside the tensor is not written. The thread that issues it commits and waits.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t from, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n\t"
               "cp.async.bulk.commit_group;" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(from), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// this thread's shared-memory stores before later reads of the async proxy (TMA)
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Instruction descriptor of the block-scaled kinds: both operands K-major, scale factor ids `id` (the byte of a 32-bit
// tensor-memory cell from which a K step's scales start), type fields, N >> 3, scale type (0 e4m3, 1 power of two), M.
__host__ __device__ constexpr uint32_t idesc_scaled(int kind, uint32_t id, uint32_t m, uint32_t n) {
  const uint32_t type = kind == 1 ? 0u : 1u;  // e4m3 is 0 among the 8-bit types, e2m1 is 1 in the 4-bit kinds
  const uint32_t pow2 = kind == 3 ? 0u : 1u;
  return id << 4 | type << 7 | type << 10 | (n >> 3) << 17 | pow2 << 23 | (m >> 7) << 27 | id << 29;
}

}  // namespace b2g

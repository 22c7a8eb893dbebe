/*
 * b2g_micro.h — C ABI of the microscaled operators (sm_100a): block-scaled 8- and 4-bit tensors, their products on the
 * tensor cores, and the layers between two products (root-mean-square norm, SiLU gate) that write such tensors.
 *
 * Conventions, return codes and error texts are those of b2g.h: device pointers are raw CUDA addresses on the current
 * device, `stream` is a cudaStream_t, every function returns B2G_OK or a negative B2G_ERR_* code with
 * b2g_last_error() text, and nothing here allocates device memory or synchronises, so every call can be captured into
 * a CUDA graph. No state is kept between calls. An output overlaps no input and no other output.
 *
 * A microscaled tensor [rows, cols] is quantised in blocks of consecutive columns (the dimension a product sums over):
 *   MXFP8  e4m3 codes, one power-of-two scale (a biased exponent byte, 255 = NaN) per 32 columns
 *   MXFP4  e2m1 codes, the same scales
 *   NVFP4  e2m1 codes, one e4m3 scale per 16 columns, one fp32 scale for the tensor
 * value = code * block scale [* tensor scale]. A block's power-of-two scale is the smallest one, from 2^-127 up, at
 * which no element passes the code's largest magnitude; an NVFP4 block's is its largest magnitude / (6 * tensor scale)
 * rounded to e4m3. Codes round to nearest, ties to even. A block that holds an infinity or a NaN gets a NaN scale. With a
 * tensor scale that is no power of two, 6 * tensor scale and block scale * tensor scale are fp32 values, and the quotients
 * by them are rounded to fp32 before they are rounded to e4m3 and to codes.
 *
 * Codes: row r starts at codes + r * pitch; MXFP8 has one byte a code, the 4-bit formats two codes a byte, the lower
 * column in the low four bits. What is left of the last byte of an odd row is zero.
 * Scales: tiles of 512 bytes for 128 rows x 4 blocks, tile (row / 128, block / 4) at
 * ((row / 128) * ceil(blocks / 4) + block / 4) * 512, byte (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4 in it:
 * the order in which the tensor cores read them. Bytes for rows and blocks that do not exist are zero.
 */
#ifndef B2G_MICRO_H_
#define B2G_MICRO_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B2G_FMT_MXFP8 1
#define B2G_FMT_MXFP4 2
#define B2G_FMT_NVFP4 3

#define B2G_VALUE_F16 0
#define B2G_VALUE_BF16 1
#define B2G_VALUE_F32 2 /* quantise and dequantise only */

typedef struct b2g_micro_tensor {
  int32_t format; /* B2G_FMT_* */
  int32_t reserved;
  int64_t rows, cols;
  void* codes;        /* 16-byte aligned */
  int64_t pitch;      /* bytes between rows: a multiple of 16 (32 for MXFP8), at least that of b2g_micro_layout */
  void* scales;       /* 16-byte aligned */
  const float* scale; /* device fp32, NVFP4 only */
} b2g_micro_tensor;

/* a strided matrix of values: element (r, c) at ptr + r * stride_r + c * stride_c (element strides) */
typedef struct b2g_micro_matrix {
  void* ptr;
  int64_t stride_r, stride_c;
} b2g_micro_matrix;

/* Smallest pitch (bytes) of a row of codes and the bytes of scales of a [rows, cols] tensor. Host only. */
int32_t b2g_micro_layout(int32_t format, int64_t rows, int64_t cols, int64_t* pitch, int64_t* scale_bytes);

/* NVFP4's scale for a whole tensor, into the device float *scale: the smallest power of two, from 2^-100 up, at which
   the largest finite magnitude is at most 6 * 448 times it. */
int32_t b2g_micro_tensor_scale(const b2g_micro_matrix* x, int64_t rows, int64_t cols, int32_t dtype, float* scale,
                               void* stream);

/* q = x, any strides. NVFP4 reads q->scale. Every byte of the codes' rows up to the pitch of b2g_micro_layout and
   every scale byte is written. */
int32_t b2g_micro_quantize(const b2g_micro_matrix* x, int32_t dtype, const b2g_micro_tensor* q, void* stream);

/* out = the values of q rounded to `dtype`, any strides. */
int32_t b2g_micro_dequantize(const b2g_micro_tensor* q, const b2g_micro_matrix* out, int32_t dtype, void* stream);

/* Product C[M, N] = A[M, K] * B[N, K]^T of two tensors of one format, fp32 accumulation, C fp16 or bf16 with unit
   column stride and row stride ldc. A plan holds the tensor maps and launch geometry for exactly these buffers on the
   current device. `status`: device int32 for bounded-wait timeouts (b2g_status_string), may be NULL. */
typedef struct b2g_micro_plan b2g_micro_plan;
int32_t b2g_micro_plan_create(const b2g_micro_tensor* a, const b2g_micro_tensor* b, void* C, int64_t ldc, int32_t dtype,
                              int32_t* status, b2g_micro_plan** out);
int32_t b2g_micro_plan_launch(const b2g_micro_plan* plan, void* stream);
int32_t b2g_micro_plan_destroy(b2g_micro_plan* plan);
/* Limit of the kernel's bounded waits, in microseconds (0: the default, one second). Plans that run as CTA pairs or split K
   over a cluster keep the default: B2G_ERR_UNSUPPORTED. A launch in which a wait runs out sets the status word; what it
   leaves in C is undefined. */
int32_t b2g_micro_plan_wait_limit(b2g_micro_plan* plan, int32_t wait_limit_us);
/* One-shot: plan, launch. */
int32_t b2g_micro_matmul(const b2g_micro_tensor* a, const b2g_micro_tensor* b, void* C, int64_t ldc, int32_t dtype,
                         int32_t* status, void* stream);

/* Product of two matrices of values, quantised on the way: C[M, N] = q(A)[M, K] * q(B)[N, K]^T, A and B of any strides and
   one type, NVFP4 with the scales of b2g_micro_tensor_scale. What quantize and matmul give one after the other, in one
   call; the quantised operands lie in `workspace`, b2g_micro_matmul_values_workspace() bytes of device memory, 16-byte
   aligned, any contents. */
int32_t b2g_micro_matmul_values_workspace(int32_t format, int64_t M, int64_t N, int64_t K, size_t* bytes);
int32_t b2g_micro_matmul_values(const b2g_micro_matrix* A, const b2g_micro_matrix* B, int64_t M, int64_t N, int64_t K,
                                int32_t value_dtype, int32_t format, void* C, int64_t ldc, int32_t dtype,
                                void* workspace, size_t workspace_bytes, int32_t* status, void* stream);

/* h = x + residual (x alone where residual is NULL); y = h * weight / sqrt(mean(h^2) + eps) by rows of `cols`. The norm
   is taken of the fp32 sum, before h is rounded; squares are summed in fp32, past whose range a row's norm is infinite.
   Outputs: h (NULL: not wanted; without a residual it is x itself and has
   to be NULL), and either y (values) or q (a
   microscaled tensor). x, residual, weight, h and y share `dtype` (F16 or BF16); weight is contiguous; cols is at most
   2^31 - 8192. */
int32_t b2g_micro_rms_norm(const b2g_micro_matrix* x, const b2g_micro_matrix* residual, const void* weight,
                           const b2g_micro_matrix* h, const b2g_micro_matrix* y, const b2g_micro_tensor* q, int64_t rows,
                           int64_t cols, float eps, int32_t dtype, void* stream);
/* Gradients: dx = r * dy * weight - h * r^3 * mean(dy * weight * h) [+ dh], r = 1 / sqrt(mean(h^2) + eps), and
   dweight = sum over rows of dy * h * r. `workspace`: b2g_micro_rms_norm_workspace() bytes of device memory, any
   contents. The sums' order is fixed for given sizes: results repeat bit for bit. */
int32_t b2g_micro_rms_norm_workspace(int64_t rows, int64_t cols, size_t* bytes);
int32_t b2g_micro_rms_norm_backward(const b2g_micro_matrix* dy, const b2g_micro_matrix* h, const void* weight,
                                    const b2g_micro_matrix* dh, const b2g_micro_matrix* dx, void* dweight,
                                    void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols, float eps,
                                    int32_t dtype, void* stream);

/* y = gate / (1 + exp(-gate)) * up of gate_up [rows, 2 cols] = [gate | up], as values (y) or microscaled (q). cols is at
   most 2^35 - 2048. */
int32_t b2g_micro_silu_mul(const b2g_micro_matrix* gate_up, const b2g_micro_matrix* y, const b2g_micro_tensor* q,
                           int64_t rows, int64_t cols, int32_t dtype, void* stream);
/* dgate_up [rows, 2 cols] from dy [rows, cols] and gate_up. */
int32_t b2g_micro_silu_mul_backward(const b2g_micro_matrix* dy, const b2g_micro_matrix* gate_up,
                                    const b2g_micro_matrix* dgate_up, int64_t rows, int64_t cols, int32_t dtype,
                                    void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B2G_MICRO_H_ */

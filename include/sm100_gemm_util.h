/*
 * C ABI of libsm100gemm_util.so: small device utilities around the GEMM plugins.
 * None of them has a counterpart in the reference (single GPU, BF16 only).
 * `stream` is a cudaStream_t; the int results are cudaError_t values (0 = success).
 */
#ifndef SM100_GEMM_UTIL_H
#define SM100_GEMM_UTIL_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* N-sharded multi-GPU run: gathered [g][M][Nb] blocks -> row-major Y[M][g*Nb].
 * elem_bytes*Nb must be a multiple of 16; pointers 16-byte aligned. */
int gemm_interleave_blocks(const void *blocked, void *Y, int g, long long M, int Nb, int elem_bytes, void *stream);

/* Idle kernel between timed launches of the reference's timing protocol: one thread calls
 * __nanosleep(us * 1000).  The reference passes 100 "ms" = 1e8 ns (sleep_kernel<<<1,1>>>(100),
 * src/common.h:16-19, 38), which the hardware cuts short at about a millisecond; us = 100000 asks for the
 * same thing. */
int gemm_spacer(unsigned us, void *stream);

/* MX scale layout (see include/sm100_gemm.h): bytes of the tiled array for `rows` rows and K
 * elements, and the conversion of a row-major [rows][K/32] ue8m0 array into it. */
size_t gemm_mx_tiled_scale_bytes(long long rows, int K);
int gemm_mx_scales_to_tiled(const void *src, void *dst, long long rows, int K, void *stream);

/* ---- quantisation kernels: the step in front of the low-precision GEMMs (device pointers, 16-byte aligned;
 * results are bit-identical to the host definitions given with each).  No reference counterpart: its
 * inputs are random bf16 in memory (src/bench.cu:353-355). */

/* bf16 x[n] -> e4m3 q[n] (round to nearest even, saturating) with one FP32 scale: *scale_out = max|x| / 448
 * (device float), q = e4m3(x * (1 / scale)).  n a multiple of 8.  amax_ws: one device float of scratch. */
int gemm_quant_e4m3_per_tensor(const void *x, void *q, float *scale_out, float *amax_ws, long long n, void *stream);

/* bf16 x[rows][K] -> MX elements + ue8m0 scales, one per 32 K-elements, written in the atom layout the GEMM
 * reads (gemm_mx_tiled_scale_bytes(rows, K) bytes; rows padded to 128 get the scale 1.0).
 * kind 8: e4m3 (MXFP8), q = rows*K bytes; kind 4: e2m1 (MX-FP4), q = rows*K/2 bytes, low nibble = even k.
 * scale code = clamp(ceil(log2(max|block| / emax)) + 127, 0, 254), 127 for a zero block; emax 448 / 6.
 * K a multiple of 128. */
int gemm_quant_mx(const void *x, void *q, void *sf_tiled, long long rows, int K, int kind, void *stream);

/* bf16 w[rows][K] -> signed int4 (two per byte, low nibble = even k) + bf16 scales [rows][K/128]:
 * s = bf16(max|group| / 7) (1 for a zero group), q = clamp(rint(w * (1 / s)), -8, 7).  K a multiple of 128. */
int gemm_quant_int4_g128(const void *w, void *q, void *scales, long long rows, int K, void *stream);

/* ---- the operators beside the projections of a decode step (csrc/token_kernels.cu).  No reference counterpart.
 * Stream-ordered, asynchronous, no allocation, no workspace; both may be captured into a CUDA graph, the first call too.
 * All pointers are device pointers of the current device.  A refused call launches nothing and returns
 * cudaErrorInvalidValue; gemm_util_last_error_message() then says why (text of the calling thread's last such call).
 * x and y are the same buffer (in place) or do not overlap. */
enum { GEMM_X_F32 = 2 };     /* beside GEMM_X_BF16 = 0 and GEMM_X_F16 = 1 of include/sm100_gemm.h */
const char *gemm_util_last_error_message(void);

/* Rotary positions on `heads` heads of each of `tokens` tokens: the pair (a, b) number i of a head becomes
 *     scale * (a cos t - b sin t,  a sin t + b cos t),   t = position * f_i          (backward: t -> -t)
 * f_i = base^(-2 i / rot_dim), scaled for contexts longer than trained (`scaling`).  Pairs: (i, i + rot_dim / 2) or
 * (2 i, 2 i + 1) of the head's first rot_dim elements; elements behind them are copied.  A token with a negative position
 * is padding: its heads are passed through unchanged.  backward = 1 turns the gradient of y into that of x (the transposed
 * map; its rows are addressed as x -> y too).  An angle is off by at most 2^-65 of a turn per position, before its sine is
 * taken (within 2^-22; 2^-20.6 for 16-bit data).
 * Strides are in elements, so that q and k are turned in place inside a fused QKV result: heads = q + k heads,
 * token stride = the row of the whole result.  Strides of x may be 0 (one head for many); heads and tokens of y do not
 * overlap. */
enum { GEMM_ROTARY_HALF = 0, GEMM_ROTARY_INTERLEAVED = 1 };
enum {
    GEMM_ROTARY_PLAIN = 0,
    GEMM_ROTARY_LINEAR = 1,  /* f_i / factor                                                                          */
    GEMM_ROTARY_NTK = 2,     /* base * factor^(rot_dim / (rot_dim - 2)) in the place of base                          */
    GEMM_ROTARY_RAMP = 3     /* f_i * w + f_i / factor * (1 - w), w = (original_length * f_i / 2 pi - low_rotations)  */
                             /* / (high_rotations - low_rotations), clamped to [0, 1]: linear in the rotations over   */
                             /* the original length.  Models whose ramp is linear in i between two pairs get other    */
                             /* frequencies from this one                                                             */
};
typedef struct GemmRotaryArgs {
    uint32_t struct_size;   /* sizeof(GemmRotaryArgs), checked                       */
    int32_t dtype;          /* GEMM_X_BF16, GEMM_X_F16 or GEMM_X_F32: type of x and y */
    int32_t layout;         /* GEMM_ROTARY_HALF / _INTERLEAVED                       */
    int32_t backward;       /* 0 / 1                                                 */
    int64_t tokens;         /* 0: nothing is done                                    */
    int32_t heads, head_dim;    /* heads * head_dim <= 2^30                              */
    int32_t rot_dim;        /* even, <= head_dim and <= 512                          */
    int32_t scaling;        /* GEMM_ROTARY_PLAIN ...                                 */
    const void *x;
    void *y;
    int64_t x_token_stride, x_head_stride, y_token_stride, y_head_stride;
    const int64_t *positions;   /* [tokens]                                          */
    double base;            /* 10000 in most models                                  */
    double factor, low_rotations, high_rotations, original_length;
    float scale;            /* multiplies cos and sin (1 when no attention scaling)  */
    int32_t reserved;       /* 0                                                     */
    void *stream;
} GemmRotaryArgs;
int gemm_rotary(const GemmRotaryArgs *args);

/* Logits of `rows` sequences before sampling, y[r][v] from x[r][v], in FP32, rounded once to the type of y:
 *     l = x;  token v in the row's history:  l = l > 0 ? l / repetition : l * repetition
 *     c = how often v was generated, c > 0:  l -= frequency * c + presence
 *     v listed in the row's biases:          l += the sum of its listed values, in the order of the list (an id that is listed
 *                                            more than once costs a walk over the row's list: fine for some hundred entries)
 *     mask bit of v is 0:                    l = -inf (whatever it was; a row that allows nothing is all -inf)
 * History: the first history_len[r] tokens of row r (at most history_ld), the first prompt_len[r] of which are the prompt:
 * they count as seen, not as generated (history_ld of 8192 or more takes a form made for long histories, whatever the lengths);
 * without a history (history NULL, a first token) no penalty applies.  Ids outside [0, vocab) are ignored, in the history and in the biases. */
typedef struct GemmLogitsArgs {
    uint32_t struct_size;   /* sizeof(GemmLogitsArgs), checked                                             */
    int32_t x_dtype, y_dtype;   /* GEMM_X_BF16, GEMM_X_F16 or GEMM_X_F32                                   */
    int32_t rows;           /* 0: nothing is done                                                          */
    int32_t vocab;          /* 1 .. 2^30                                                                   */
    int32_t reserved;       /* 0                                                                           */
    const void *x;
    void *y;
    int64_t x_ld, y_ld;     /* row pitches in elements, >= vocab                                           */
    const int32_t *history; /* [rows][history_ld], or NULL                                                 */
    int64_t history_ld;     /* < 2^29                                                                      */
    const int32_t *history_len;     /* [rows], with history                                                */
    const int32_t *prompt_len;      /* [rows], or NULL: everything was generated                           */
    const float *repetition, *presence, *frequency;     /* [rows] each, or NULL: 1, 0, 0                   */
    const int32_t *bias_ids;        /* biases of row r: entries bias_begin[r] .. bias_begin[r + 1] - 1     */
    const float *bias_values;
    const int32_t *bias_begin;      /* [rows + 1], not decreasing, or NULL (all three)                     */
    const uint32_t *mask;   /* [rows][mask_ld], bit v % 32 of word v / 32: 1 = allowed; or NULL            */
    int64_t mask_ld;        /* >= ceil(vocab / 32)                                                         */
    void *stream;
} GemmLogitsArgs;
int gemm_logits(const GemmLogitsArgs *args);

/* ---- offline weight packing and the weight file (host memory, host code).  No reference counterpart. */
enum {
    GEMM_FILE_ERR_ARG = -5,      /* null pointer, value out of range, K not a multiple the layout needs */
    GEMM_FILE_ERR_CHECKSUM = -4, /* payload does not match the header's checksum                         */
    GEMM_FILE_ERR_SIZE = -3,     /* caller buffer too small                                              */
    GEMM_FILE_ERR_FORMAT = -2,   /* not a weight file of this version, or truncated                      */
    GEMM_FILE_ERR_IO = -1        /* open / read / write / rename failed                                  */
};

/* First bytes of a weight file (the header block is padded to 256 bytes; payloads start on 256-byte
 * boundaries: elements at 256, scales at 256 + round_up(elem_bytes, 256)). */
typedef struct GemmWeightFileInfo {
    char magic[8];        /* "SM100QW\0"                                                    */
    uint32_t version;     /* 1                                                              */
    uint32_t dtype;       /* GEMM_DT_* of include/sm100_gemm.h                              */
    uint32_t layout;      /* version of the element / scale layouts (1 = those of sm100_gemm.h) */
    uint32_t group;       /* K-elements per scale: 32 (MX kinds), 128 (W4A16), 0 (none)     */
    uint64_t N, K;        /* weight rows (output columns) and reduction length              */
    uint64_t elem_bytes, scale_bytes;
    float tensor_scale;   /* FP8 per-tensor scale, 1 elsewhere                              */
    uint32_t checksum;    /* FNV-1a (32 bit) over the element payload, then the scale payload */
} GemmWeightFileInfo;

/* Bytes of the element / scale payload of an N x K weight matrix of the given GEMM_DT_*. */
size_t gemm_packed_weight_bytes(int dtype, long long N, int K);
size_t gemm_packed_scale_bytes(int dtype, long long N, int K);

/* int4 values in [-8, 7], one per int8, row-major -> two per byte (low nibble = even k), and back. */
int gemm_pack_int4_host(const int8_t *q, long long N, int K, uint8_t *out);
int gemm_unpack_int4_host(const uint8_t *packed, long long N, int K, int8_t *q);
/* e2m1 codes 0..15, one per byte -> two per byte (low nibble = even k), and back. */
int gemm_pack_fp4_host(const uint8_t *codes, long long N, int K, uint8_t *out);
int gemm_unpack_fp4_host(const uint8_t *packed, long long N, int K, uint8_t *codes);
/* row-major ue8m0 scales [rows][K/32] <-> the 512-byte atom layout (host version of gemm_mx_scales_to_tiled). */
int gemm_mx_scales_to_tiled_host(const uint8_t *src, long long rows, int K, uint8_t *dst);
int gemm_mx_scales_from_tiled_host(const uint8_t *src, long long rows, int K, uint8_t *dst);

/* Writes / inspects / reads a weight file.  `elems` and `scales` are already in the packed layouts (sizes
 * from the two functions above; scales NULL when the type has none).  The file is written under a temporary
 * name and renamed.  read() fills caller buffers and verifies the checksum.  0 or a GEMM_FILE_ERR_*. */
int gemm_weight_file_write(const char *path, int dtype, long long N, int K, float tensor_scale, const void *elems, const void *scales);
int gemm_weight_file_info(const char *path, GemmWeightFileInfo *out);
int gemm_weight_file_read(const char *path, void *elems, size_t elem_capacity, void *scales, size_t scale_capacity);

#ifdef __cplusplus
}
#endif
#endif /* SM100_GEMM_UTIL_H */

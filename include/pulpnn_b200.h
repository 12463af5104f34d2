/*
 * pulpnn_b200.h -- C ABI of the B200 (sm_100a) implementation of the PULP-NN
 * 8-bit HWC inference kernels.
 *
 * Every kernel entry point keeps the name, the parameter list and the
 * arithmetic of the reference prototype it replaces; the citation beside each
 * one is the line of 32bit/include/pulp_nn_kernels.h (the 64bit/ header is
 * identical except that k/lambda are int64_t). The reference ships two source
 * trees that export the same names with different batch-norm widths; here one
 * library exports both, suffixed _bn32 / _bn64 (libpulpnn_b200.so), and two
 * thin libraries (libpulpnn_b200_32.so, libpulpnn_b200_64.so, see
 * pulpnn_b200_dropin.h) export the unsuffixed reference names.
 *
 * Calling convention on the GPU
 *  - ONE host thread makes the call once; the grid plays the role of the
 *    reference's cluster of cores. Work is enqueued on the calling thread's
 *    current stream (pulpnn_set_stream) and the call returns without waiting,
 *    unless a buffer is in host memory (see below).
 *  - Pointers may be device pointers (the fast path) or ordinary host
 *    pointers. Host buffers are staged through device memory owned by the
 *    library and the call then returns only after the results are back in the
 *    caller's buffers.
 *  - The reference processes one image per call. pulpnn_set_batch(n) makes
 *    every activation pointer address n images stored back to back; weights
 *    and batch-norm parameters are shared by the batch.
 *  - Scratch arguments of the reference (pIm2ColBuffer, bufferC, bufferB) are
 *    accepted and ignored; they may be NULL.
 *  - The entry points return void like the reference. A call whose arguments
 *    are invalid or outside the supported domain enqueues nothing and records
 *    an error for the calling thread (pulpnn_last_error). There is no CPU
 *    fallback of any kind.
 */
#ifndef PULPNN_B200_H
#define PULPNN_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status ------------------------------------------------------------- */
enum {
  PULPNN_OK = 0,
  PULPNN_ERR_INVALID_ARG = 1,   /* NULL pointer, zero dimension, shift out of range ...     */
  PULPNN_ERR_UNSUPPORTED = 2,   /* outside the domain where the reference is well defined   */
  PULPNN_ERR_CUDA = 3,          /* a CUDA runtime/driver call failed                        */
  PULPNN_ERR_NO_DEVICE = 4,     /* no usable GPU: the library never computes on the CPU     */
  PULPNN_ERR_DEVICE_WAIT = 5    /* a bounded wait inside a kernel ran out (see status word) */
};

/* ---- per-thread context -------------------------------------------------- */
int  pulpnn_set_device(int device);          /* also creates the context; returns a status   */
int  pulpnn_set_stream(void *cuda_stream);   /* cudaStream_t; NULL = the default stream       */
int  pulpnn_set_batch(int n_images);         /* n >= 1; sticky until changed                  */
int  pulpnn_get_batch(void);
int  pulpnn_synchronize(void);               /* waits for the stream; returns a status        */
int  pulpnn_last_error(void);
const char *pulpnn_last_error_message(void);
void pulpnn_clear_error(void);
/* kernels launched by this library since it was loaded (all threads) */
unsigned long long pulpnn_launch_count(void);
/* The kernel family of the calling thread's latest launch ("igemm_tc_kernel", ...), "" before the first:
 * which of the kernels that serve an entry point a call took, for tests and measurements. */
const char *pulpnn_last_kernel(void);
/* Reads and clears the device-side status word: 0 = every bounded wait in the
 * tensor-core kernels completed. Synchronises the stream first. */
int  pulpnn_device_status(void);

/* Tuning / test switches (value 0 or 1 unless stated). */
enum {
  PULPNN_OPT_FORCE_GENERIC = 1,   /* route contractions to the generic CUDA-core kernel      */
  PULPNN_OPT_MAXPOOL_CLOBBER = 2, /* also reproduce the reference's overwrite of Im_in       */
  PULPNN_OPT_SPLIT_K = 3,         /* 0 = choose automatically, n > 0 = force n K-slices      */
                                  /* (pulpnn_attn_decode: n CTAs for a sequence)             */
  PULPNN_OPT_FUSE_DWPW = 4,       /* network runner: run a 3x3 stride-1 depthwise layer and   */
                                  /* the pointwise layer behind it as ONE kernel where a      */
                                  /* fused kernel exists (default 1); results are identical   */
  PULPNN_OPT_TUNE = 5             /* measurement switch, a bit mask (0 = the defaults). Bits 3-5 */
                                  /* select alternative launch configurations (8: SM-pair GEMM   */
                                  /* from K = 512 on, 16: no few-rows GEMM, 32: the 32-channel   */
                                  /* fused pair with its depthwise sums on the tensor cores);    */
                                  /* results identical.                                          */
                                  /* Bits 8-11 switch PARTS of the tensor-core kernels off to    */
                                  /* time the rest (epilogue, loads, MMAs, stores): the output   */
                                  /* is then wrong by design. Never set them outside a timing run */
};
int  pulpnn_set_option(int option, int value);
int  pulpnn_get_option(int option);

/* ---- kernel entry points -------------------------------------------------- */
/* shared parameter list of the convolution family (pulp_nn_kernels.h:56-82) */
#define PULPNN_CONV_PARAMS(BN_T)                                                              \
  const uint8_t *pInBuffer, uint8_t *pIm2ColBuffer, const int8_t *bias, uint8_t *pOutBuffer,  \
  const int8_t *pWeight, BN_T *k, BN_T *lambda, const uint16_t out_mult,                      \
  const uint16_t out_shift, const uint16_t dim_in_x, const uint16_t dim_in_y,                 \
  const uint16_t ch_in, const uint16_t dim_out_x, const uint16_t dim_out_y,                   \
  const uint16_t ch_out, const uint16_t dim_kernel_x, const uint16_t dim_kernel_y,            \
  const uint16_t padding_y_top, const uint16_t padding_y_bottom,                              \
  const uint16_t padding_x_left, const uint16_t padding_x_right, const uint16_t stride_x,     \
  const uint16_t stride_y, int flag_relu, int flag_batch_norm

/* parameter list of the depthwise family (pulp_nn_kernels.h:282-309) */
#define PULPNN_DW_PARAMS(BN_T)                                                                \
  const uint8_t *Im_in, uint8_t *bufferC, const int8_t *bias, uint8_t *Im_out,                \
  const int8_t *wt, uint8_t *bufferB, BN_T *k, BN_T *lambda, uint16_t out_mult,               \
  uint16_t out_shift, const uint16_t dim_im_in_x, const uint16_t dim_im_in_y,                 \
  const uint16_t ch_im_in, const uint16_t dim_im_out_x, const uint16_t dim_im_out_y,          \
  const uint16_t ch_im_out, const uint16_t dim_kernel_x, const uint16_t dim_kernel_y,         \
  const uint16_t padding_y_top, const uint16_t padding_y_bottom,                              \
  const uint16_t padding_x_left, const uint16_t padding_x_right, const uint16_t stride_x,     \
  const uint16_t stride_y, int8_t FLAG_RELU, int8_t FLAG_BATCH_NORM

/* parameter list of the pooling pair (pulp_nn_kernels.h:264-280 and :33-53) */
#define PULPNN_POOL_GEOMETRY                                                                  \
  uint16_t dim_im_in_x, uint16_t dim_im_in_y, uint16_t ch_im_in, uint16_t dim_im_out_x,       \
  uint16_t dim_im_out_y, uint16_t dim_kernel_x, uint16_t dim_kernel_y, uint16_t padding_t,    \
  uint16_t padding_b, uint16_t padding_l, uint16_t padding_r, uint16_t stride_x,              \
  uint16_t stride_y

/*
 * One tree of entry points. SFX is appended to every reference name, BN_T is
 * the batch-norm parameter type of that tree.
 *
 *  pulp_nn_conv_Ho_parallel         pulp_nn_kernels.h:56    zero-padded convolution, HWC in/out,
 *  pulp_nn_conv_HoWo_parallel       pulp_nn_kernels.h:112   weights [ch_out][ky][kx][ch_in]; the two
 *                                                           differ in the reference only in how cores
 *                                                           split the rows, so they share one kernel
 *  pulp_nn_pointwise_HoWo_parallel  pulp_nn_kernels.h:140   1x1 convolution; kernel/pad/stride
 *                                                           arguments are ignored as in the reference
 *  pulp_nn_conv_Co_parallel         pulp_nn_kernels.h:84    the remaining core-slicing variants: the
 *  pulp_nn_pointwise_Ho_parallel    pulp_nn_kernels.h:168   same function of the same arguments as
 *  pulp_nn_pointwise_Co_parallel    pulp_nn_kernels.h:196   the two above (a grid has no cores to
 *                                                           slice over), so they share their kernels.
 *                                                           Defined as the convolution itself: the
 *                                                           reference's Co-parallel files mis-step
 *                                                           their bias and weight pointers between
 *                                                           channel chunks, which is not imitated
 *  pulp_nn_depthwise_generic        pulp_nn_kernels.h:282   CHW in, HWC out
 *  pulp_nn_depthwise_generic_less_4_weights  :311           same, for kernels of fewer than 4 taps
 *                                                           (accepts any number of taps)
 *  pulp_nn_depthwise_3x3_s1         pulp_nn_kernels.h:340   CHW in (R x C), HWC out (R-2 x C): 3x3,
 *                                                           stride 1, no vertical padding, no bias.
 *                                                           Accepted for p_l = p_r = 1 and even C,
 *                                                           where the reference is a zero-padded
 *                                                           convolution; memory_chan is ignored
 *  pulp_nn_matmul                   pulp_nn_kernels.h:248   the convolutions' inner kernel: two
 *                                                           im2col columns (pInBuffer, pInBuffer +
 *                                                           num_col_im2col) x ch_out filters into
 *                                                           pOut and pOut2; returns pOut + 2*ch_out.
 *                                                           The batch setting does not apply
 *  pulp_nn_linear                   pulp_nn_kernels.h:224   uint8 output, requantised
 *  pulp_nn_linear_out_32            pulp_nn_kernels.h:239   raw int32 output; bias is read as int32[]
 *  pulp_nn_maxpool                  pulp_nn_kernels.h:264   Im_in is left intact unless
 *                                                           PULPNN_OPT_MAXPOOL_CLOBBER is set
 *  pulp_nn_avgpool                  pulp_nn_kernels.h:33    lambda/out_add have the tree's width
 *  pulp_nn_add                      pulp_nn_kernels.h:21
 *
 *  pulpnn_depthwise_hwc             extension: pulp_nn_depthwise_generic arithmetic on HWC input
 *                                   (what every producer in this API emits); no reference counterpart
 */
#define PULPNN_DECLARE_TREE(SFX, BN_T)                                                        \
  void pulp_nn_conv_Ho_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                               \
  void pulp_nn_conv_HoWo_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                             \
  void pulp_nn_pointwise_HoWo_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                        \
  void pulp_nn_conv_Co_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                               \
  void pulp_nn_pointwise_Ho_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                          \
  void pulp_nn_pointwise_Co_parallel##SFX(PULPNN_CONV_PARAMS(BN_T));                          \
  void pulp_nn_depthwise_generic##SFX(PULPNN_DW_PARAMS(BN_T));                                \
  void pulp_nn_depthwise_generic_less_4_weights##SFX(PULPNN_DW_PARAMS(BN_T));                 \
  void pulpnn_depthwise_hwc##SFX(PULPNN_DW_PARAMS(BN_T));                                     \
  void pulp_nn_depthwise_3x3_s1##SFX(uint8_t *In_Img, uint8_t *Out_Img, int R, int C, int CH,  \
                                     int p_l, int p_r, int8_t *Kernel, int8_t out_shift,      \
                                     uint16_t out_mult, BN_T *kappa, BN_T *lambda,            \
                                     int flag_relu, int flag_batch_norm,                      \
                                     unsigned int *memory_chan);                              \
  uint8_t *pulp_nn_matmul##SFX(const int8_t *pWeight, uint8_t *pInBuffer, uint16_t ch_out,    \
                               uint16_t num_col_im2col, uint16_t out_shift, uint16_t out_mult,\
                               BN_T *k, BN_T *lambda, const int8_t *bias, uint8_t *pOut,      \
                               uint8_t *pOut2, int flag_relu, int flag_batch_norm);           \
  void pulp_nn_linear##SFX(uint8_t *pInBuffer, int8_t *bias, uint8_t *pOutBuffer,             \
                           int8_t *pWeights, BN_T *k, BN_T *lambda, uint16_t out_mult,        \
                           int8_t out_shift, uint16_t dim_vec, uint16_t num_o_neurons,        \
                           int flag_relu, int flag_batch_norm);                               \
  void pulp_nn_linear_out_32##SFX(uint8_t *pInBuffer, int8_t *bias, int32_t *pOutBuffer,      \
                                  int8_t *pWeights, uint16_t dim_vec, uint16_t num_o_neurons);\
  void pulp_nn_maxpool##SFX(uint8_t *Im_in, uint8_t *Im_out, PULPNN_POOL_GEOMETRY);           \
  void pulp_nn_avgpool##SFX(uint8_t *Im_in, uint8_t *Im_out, BN_T lambda, uint16_t out_shift, \
                            BN_T out_add, PULPNN_POOL_GEOMETRY, int flag_requant);            \
  void pulp_nn_add##SFX(uint8_t *Im_in_1, uint8_t *Im_in_2, uint8_t *Im_out,                  \
                        uint16_t out_mult1, uint16_t out_mult2, uint16_t out_shift,           \
                        uint16_t dim_im_in_h, uint16_t dim_im_in_w, uint16_t ch_im_in);

PULPNN_DECLARE_TREE(_bn32, int32_t)
PULPNN_DECLARE_TREE(_bn64, int64_t)

/*
 * Layout change of uint8 activations, CHW <-> HWC, for the images of the current batch. No
 * counterpart in the reference, which needs one all the same: pulp_nn_depthwise_generic reads CHW
 * (32bit/src/pulp_nn_depthwise_generic.c:74) while every kernel of the library, the depthwise one
 * included, writes HWC (ibid. :81,179). In and out must not overlap.
 */
void pulpnn_chw_to_hwc(const uint8_t *Im_in, uint8_t *Im_out, uint16_t dim_im_x, uint16_t dim_im_y, uint16_t ch_im);
void pulpnn_hwc_to_chw(const uint8_t *Im_in, uint8_t *Im_out, uint16_t dim_im_x, uint16_t dim_im_y, uint16_t ch_im);

/*
 * Sub-byte unpack helpers of the reference as bulk device operations. Packed values sit
 * little-endian in their bytes (element i of a byte = bits [w*i, w*i+w)).
 *   pulp_nn_im2col_u4_to_u8, pulp_nn_im2col_u2_to_u8   32bit/include/pulp_nn_utils.h:65,67
 *       (32bit/src/pulp_nn_utils.c:396-438): blockSize = number of uint8 results; it must be a
 *       multiple of 2 (4): the reference's tail loops never end otherwise.
 *   pulpnn_i4_to_i8, pulpnn_i2_to_i8                    the sign-extending counterparts, bulk forms of
 *       pulp_nn_i4_to_i8 / pulp_nn_i2_to_i8 (pulp_nn_utils.c:255,289); n = number of int8 results.
 * Device or host buffers; the batch setting does not apply.
 */
void pulp_nn_im2col_u4_to_u8(uint8_t *pInput, uint8_t *pOutput, unsigned int blockSize);
void pulp_nn_im2col_u2_to_u8(uint8_t *pInput, uint8_t *pOutput, unsigned int blockSize);
void pulpnn_i4_to_i8(const int8_t *pSrc, int8_t *pDst, unsigned int n);
void pulpnn_i2_to_i8(const int8_t *pSrc, int8_t *pDst, unsigned int n);

/*
 * The scalar requantisers of pulp_nn_utils.h as element-wise bulk device operations: n int32
 * accumulators in, one result byte each out (not packed); element i takes the parameters of channel
 * i % channels; bits = 8, 4 or 2 selects the clip range 255 / 15 / 3. Device or host buffers.
 *   pulpnn_bn_quant_bulk     pulp_nn_bn_quant_u8 / _u4 / _u2   32bit/include/pulp_nn_utils.h:23,29,41
 *                            (32bit/src/pulp_nn_utils.c:35-45,158-167,180-189): clip((k*phi + lambda) >> d),
 *                            int32 wrap-around in the 32-bit tree, int64 in the 64-bit tree
 *   pulpnn_quant_bulk        pulp_nn_quant_u8 / _u4 / _u2      pulp_nn_utils.h:25,31,43
 *                            (pulp_nn_utils.c:148-156,169-178,191-199): clip((m*phi) >> d); the shifted
 *                            value is cut to int16 for 8 bits in both trees and for 4 / 2 bits in the
 *                            64-bit tree only (64bit/src/pulp_nn_utils.c:153,175,197)
 *   pulpnn_threshold_quant_bulk   pulp_nn_i4_quant / pulp_nn_i2_quant   pulp_nn_utils.h:69,71
 *                            (pulp_nn_utils.c:438-540): the signed 4- or 2-bit level of each input among a
 *                            channel's thresholds (int16; 16 per channel of which 15 are read for 4
 *                            bits, 4 per channel of which 3 are read for 2 bits), one int8 out
 *   pulp_nn_avg_and_replace_int8   pulp_nn_utils.h:39 (pulp_nn_utils.c:95-115), the reference's own
 *                            signature: base[i] = (base[i] + target[i]) >> 1 on signed bytes, for
 *                            length >> 2 whole words; the batch setting does not apply
 */
void pulpnn_bn_quant_bulk_bn32(const int32_t *phi, const int32_t *k, const int32_t *lambda, int8_t d, uint8_t *out,
                               unsigned int n, unsigned int channels, int bits);
void pulpnn_bn_quant_bulk_bn64(const int32_t *phi, const int64_t *k, const int64_t *lambda, int8_t d, uint8_t *out,
                               unsigned int n, unsigned int channels, int bits);
void pulpnn_quant_bulk_bn32(const int32_t *phi, int16_t m, int8_t d, uint8_t *out, unsigned int n, int bits);
void pulpnn_quant_bulk_bn64(const int32_t *phi, int16_t m, int8_t d, uint8_t *out, unsigned int n, int bits);
void pulpnn_threshold_quant_bulk(const int32_t *in, const int16_t *thr, int8_t *out, unsigned int n,
                                 unsigned int channels, int bits);
void pulp_nn_avg_and_replace_int8(int8_t *base, int8_t *target, uint16_t length);

/*
 * pulpnn_linear_out_32_static_scratch -- no counterpart in the reference.
 *
 * The arithmetic of pulp_nn_linear_out_32 (int32 accumulators, bias read as int32 words, no
 * requantisation) for n_vectors input vectors, computed with K split over k_slices groups of
 * CTAs, for callers that must not allocate: a service that has given all free device memory to
 * its own pool, or a deployment with a fixed, audited memory budget, cannot have a library call
 * cudaMalloc behind its back (the ordinary split-K path does, the first time and whenever a
 * larger problem arrives). Here the partial sums live in a 4 MiB array that is part of the
 * library image (every GPU that loads the library holds it until the process exits), and the
 * call uses no cudaMalloc, cudaFree or any other allocating routine.
 *
 *  - All four buffers must be device (or managed) memory of the context's GPU -- host buffers
 *    would need staging memory; pInBuffer and pWeights 16-byte aligned, pOutBuffer and bias
 *    4-byte aligned; bias may be NULL; dim_vec must be a multiple of 16.
 *  - Limit: k_slices * n_vectors * num_o_neurons <= 1048576 partial sums (k_slices >= 2, and
 *    dim_vec long enough to split); anything larger is refused with PULPNN_ERR_UNSUPPORTED.
 *  - The first call on a device looks up the array's device address; make that first call
 *    before any stream capture is begun.
 *  - Every call shares the one array, which keeps the previous call's contents. Nothing in it
 *    has to start at zero (each call writes every partial sum it later reads), but two calls
 *    whose kernels overlap on the GPU -- different streams, different host threads -- race.
 *  - Enqueues on the calling thread's stream and returns a status (PULPNN_OK or an error code).
 *  - A bounded wait that runs out inside its kernel is recorded in a status word that is built
 *    into the library as well, and shows up in pulpnn_device_status() like any other.
 */
int pulpnn_linear_out_32_static_scratch(const uint8_t *pInBuffer, const int32_t *bias,
                                        int32_t *pOutBuffer, const int8_t *pWeights, int dim_vec,
                                        int num_o_neurons, int n_vectors, int k_slices);

/*
 * pulpnn_selftest_wait_timeout -- diagnostic, no counterpart in the reference.
 *
 * Every wait inside the TMA / tensor-core kernels is bounded: when it runs out the kernel leaves
 * through its ordinary exit and records a code in the device status word. This call exercises
 * exactly that path without disturbing anything: a one-warp kernel waits, with the given limit
 * (microseconds, clamped to 1..100000), on a barrier that nothing will ever complete. After it,
 * pulpnn_device_status() returns a non-zero code (and clears it) and pulpnn_last_error() is
 * PULPNN_ERR_DEVICE_WAIT; the GPU and the context stay usable. Returns PULPNN_OK when the
 * kernel was enqueued.
 */
int pulpnn_selftest_wait_timeout(unsigned int limit_us);

/* ---- attention over a paged cache of keys and values -------------------------
 * What a decoder built on the 8-bit fully connected layers runs between them; no counterpart in the
 * reference. pulp_nn_linear_out_32's accumulators become rotated queries and cached keys and values
 * (pulpnn_kv_append), one new token per sequence reads the cache (pulpnn_attn_decode), a prompt is
 * attended to as a whole (pulpnn_attn_prompt), cached rows come back as 16-bit rows (pulpnn_kv_gather),
 * and both attentions can write the uint8 activations that pulp_nn_linear reads.
 *
 *  - Each call enqueues ONE kernel (pulpnn_attn_decode at most two) on the calling thread's stream, returns
 *    a status (PULPNN_OK or an error code, also recorded for pulpnn_last_error) and may be captured
 *    into a CUDA graph. The batch setting does not apply.
 *  - Every buffer is device (or managed) memory of the context's GPU. Strides count elements and, but for
 *    pulpnn_attn_prompt's, may be negative; the channels of a row lie side by side, and rows of queries, keys, values and outputs begin on 16-byte boundaries (uint8
 *    outputs of the attentions: on 4-byte ones).
 *  - head_dim: a multiple of 8 up to 128; of 16 where the cache holds 8 bits.
 *  - A wait inside a kernel that runs out leaves that call's rows void and shows in pulpnn_device_status(), unless the
 *    call was captured ahead of all its thread's calls outside a capture: then there is no word yet to report into.
 *  - Sizes come from the host; slots, positions, block tables, lengths and offsets are read from device
 *    memory when the kernel runs. Values among them that point outside the buffers read and write nothing:
 *    what each call does instead stands beside it.
 */
enum {
  PULPNN_TYPE_F16 = 0, PULPNN_TYPE_BF16 = 1, PULPNN_TYPE_F32 = 2, PULPNN_TYPE_S32 = 3, PULPNN_TYPE_S8 = 4,
  PULPNN_TYPE_U8 = 5
};

/* Keys and values in pages of page_size slots. Element (slot s, head h, channel c) of the keys is
 * k[(s / page_size) * page_stride + (s % page_size) * slot_stride + h * head_stride + c]; the values and, for
 * PULPNN_TYPE_S8, the scales (one float per slot and head) likewise. type: F16, BF16 or S8; an S8 row stands for
 * code * scale, and a scale that is NaN makes its row NaN. */
typedef struct {
  void *k, *v;
  float *k_scale, *v_scale;                 /* NULL unless type is PULPNN_TYPE_S8 */
  int64_t page_stride, slot_stride, head_stride;
  int64_t scale_page_stride, scale_slot_stride, scale_head_stride;
  int32_t type, n_pages, page_size, n_heads, head_dim, reserved;
} pulpnn_kv_cache_t;

/*
 * pulpnn_kv_append -- rotates queries and keys, and stores keys and values into the cache.
 *
 * Token t of head h: x = in (F16, BF16, F32) or in * step[h * head_dim + c] (S32). The first rotary_dim channels of
 * q and k turn by the angle positions[t] * inv_freq[i], i < rotary_dim / 2: (a, b) -> (a cos - b sin,
 * b cos + a sin) of the channels (i, i + rotary_dim / 2), or (2i, 2i + 1) where interleaved is set. The angle is
 * computed in 64 bits; its part of a turn is then rounded to 24 bits. q_out receives q; row slots[t] of the cache receives k
 * and v, rounded to its 16-bit type, or as S8 codes: the whole numbers nearest to x * (127 / max|x|) in 32 bits (within 2^-15
 * of halfway between two of them, either), with the scale max|x| / 127 (rows below 2^-100 become 0; a row with a NaN or an
 * infinity gets the scale NaN). k_out and v_out (may be NULL) receive the rows before they are cut to 8 bits.
 *
 *  - in_type: F16, BF16, F32 or S32. out_type: F16 or BF16, of q_out, k_out and v_out, whatever the cache holds.
 *  - q may be NULL (with q_out); positions and inv_freq may be NULL where rotary_dim is 0 (even, at most head_dim).
 *  - q_out may be q (k_out k, v_out v) with the same strides and a type of the same size; other overlaps are undefined.
 *  - A token whose slot lies outside the cache (-1: padding) is not stored; its q_out, k_out, v_out are written.
 *    Slots of one call differ: what a slot that two tokens name holds afterwards is undefined.
 */
typedef struct {
  const void *q, *k, *v;                    /* [n_tokens][heads][head_dim] */
  void *q_out, *k_out, *v_out;
  const float *q_step, *k_step, *v_step;    /* [heads * head_dim], S32 only */
  const int64_t *slots;                     /* [n_tokens] */
  const int32_t *positions;                 /* [n_tokens] */
  const double *inv_freq;                   /* [rotary_dim / 2], radians per position */
  int64_t q_stride[2], k_stride[2], v_stride[2];             /* token, head */
  int64_t q_out_stride[2], k_out_stride[2], v_out_stride[2];
  int32_t n_tokens, n_q_heads, rotary_dim, interleaved, in_type, out_type;
} pulpnn_kv_append_t;
int pulpnn_kv_append(const pulpnn_kv_cache_t *cache, const pulpnn_kv_append_t *args);

/*
 * pulpnn_kv_gather -- rows slots[0 .. n_tokens) of the cache as 16-bit rows (S8: code * scale in 32 bits, then rounded). A slot
 * outside the cache gives a row of zeros. out_type: F16 or BF16; a 16-bit cache has the same. k_out or v_out may be NULL.
 */
typedef struct {
  const int64_t *slots;                     /* [n_tokens] */
  void *k_out, *v_out;                      /* [n_tokens][n_heads][head_dim] */
  int64_t k_out_stride[2], v_out_stride[2]; /* token, head */
  int32_t n_tokens, out_type;
} pulpnn_kv_gather_t;
int pulpnn_kv_gather(const pulpnn_kv_cache_t *cache, const pulpnn_kv_gather_t *args);

/*
 * pulpnn_attn_decode -- attention of one new token per sequence over the cache:
 * out[b][h] = sum over t of softmax(scale * q[b][h] . k[t]) v[t], where t runs over tokens 0 .. seq_lens[b] - 1 of
 * sequence b (the last `window` of them where window > 0), token t lies in slot t % page_size of page
 * block_table[b * table_stride + t / page_size], and query head h reads key head h / (n_heads / cache heads).
 * lse (may be NULL, [n_seqs][n_heads]) receives the natural logarithm of the softmax's sum. A sequence without tokens
 * gives zeros, and minus infinity in lse.
 *
 *  - q_type: F16 or BF16, the cache's where that is 16 bits wide. out_type: q_type, or U8: out * (1 / out_step) in 32 bits,
 *    rounded to the nearest, plus out_zero, cut to 0 .. 255; a NaN gives out_zero.
 *  - out overlaps no input. A long sequence of a call with few of them is read by several groups of CTAs, whose sums are
 *    joined by a second kernel through memory allocated in the stream's order (in a capture: owned by the graph).
 *  - Lengths are cut to 0 .. max_pages * page_size. A token whose page lies outside the cache is left out, as if masked.
 *    How many CTAs share a sequence goes by max_pages, since lengths are not known on the host: a table much wider than the
 *    sequences costs time (64 of 1000 tokens: 51 us, 75 with a table for 131072).
 *  - Scores, sums and the softmax are held in 32 bits; a token's weight is rounded to q_type for its product with v. fp16
 *    weights are off by 2^-32 of the largest at most where that is more than half a step.
 *  - S8 caches: the weight times the value's scale is what is rounded, to fp16, and q is, after a power of two that brings its
 *    largest value to 1 .. 2: bf16 queries lose what lies below 2^-24 of that.
 */
typedef struct {
  const void *q;                            /* [n_seqs][n_heads][head_dim] */
  void *out;
  float *lse;
  const int32_t *block_table, *seq_lens;    /* [n_seqs][max_pages], [n_seqs] */
  int64_t q_stride[2], out_stride[2], table_stride;          /* sequence, head */
  float scale, out_step;
  int32_t out_zero, q_type, out_type, n_seqs, n_heads, max_pages, window, reserved;
} pulpnn_attn_decode_t;
int pulpnn_attn_decode(const pulpnn_kv_cache_t *cache, const pulpnn_attn_decode_t *args);

/*
 * pulpnn_attn_prompt -- attention over whole prompts, packed one behind the other: sequence b holds rows cu_q[b] ..
 * cu_q[b + 1] - 1 of q and out and rows cu_k[b] .. cu_k[b + 1] - 1 of k and v; query head h reads key head
 * h / (n_heads / n_kv_heads). Query i of a sequence of Lq queries and Lk keys has the position i + Lk - Lq (keys that
 * lie before a prompt's first query are its cached beginning). causal: it sees the keys 0 .. position; window > 0
 * (causal only): the last `window` of these. lse as above, [n_q_rows][n_heads]. A query that sees no key gives zeros, and
 * minus infinity in lse.
 *
 *  - type: F16 or BF16, of q, k and v. out_type: type, or U8 as above. scale > 0.
 *  - What a query does not see does not reach its result, infinities and NaN there included.
 *  - out overlaps no input; strides are positive and below 2^38. Offsets ascend; what lies beyond the rows there are is cut
 *    off, and a sequence that ends before it begins is empty. Rows of out and lse that no sequence holds are left as
 *    they were. At most 2^24 sequences, and 2^26 of sequences times query heads.
 *  - Scores, sums and the softmax are held in 32 bits; weights are rounded to `type` for their product with v (fp16 weights: off
 *    by 2^-30 of the largest at most where that is more than half a step). lse: its logarithm is off by 2^-22 or 2 units in
 *    its last place.
 */
typedef struct {
  const void *q, *k, *v;                    /* [rows][heads][head_dim] */
  void *out;
  float *lse;
  const int32_t *cu_q, *cu_k;               /* [n_seqs + 1] */
  int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];      /* row, head */
  float scale, out_step;
  int32_t out_zero, type, out_type, n_q_rows, n_k_rows, n_seqs, n_heads, n_kv_heads, head_dim, causal, window, reserved;
} pulpnn_attn_prompt_t;
int pulpnn_attn_prompt(const pulpnn_attn_prompt_t *args);

/* ---- sequential network runner --------------------------------------------
 * The reference is a kernel library; its user chains the calls. This runner is
 * that chain for one GPU: layers are appended in order, parameters are copied
 * to the device once, and run() pushes a batch through every layer with
 * activations ping-ponging between two device buffers owned by the network.
 * Depthwise layers use the HWC-input kernel, so no layout change is needed
 * between layers. Different GPUs run different slices of the batch; nothing is
 * exchanged between them.
 */
typedef struct pulpnn_net pulpnn_net_t;

enum {
  PULPNN_LAYER_CONV = 0,        /* pulp_nn_conv_Ho_parallel                       */
  PULPNN_LAYER_POINTWISE = 1,   /* pulp_nn_pointwise_HoWo_parallel                */
  PULPNN_LAYER_DEPTHWISE = 2,   /* pulpnn_depthwise_hwc                            */
  PULPNN_LAYER_AVGPOOL = 3,     /* pulp_nn_avgpool, flag_requant = 0              */
  PULPNN_LAYER_MAXPOOL = 4,     /* pulp_nn_maxpool                                */
  PULPNN_LAYER_LINEAR_OUT_32 = 5/* pulp_nn_linear_out_32 (must be the last layer) */
};

typedef struct {
  int type;                       /* PULPNN_LAYER_*                                     */
  int dim_in_x, dim_in_y, ch_in;
  int dim_out_x, dim_out_y, ch_out;
  int dim_kernel_x, dim_kernel_y;
  int padding_y_top, padding_y_bottom, padding_x_left, padding_x_right;
  int stride_x, stride_y;
  int out_mult, out_shift, flag_relu, flag_batch_norm;
  const int8_t *weights;          /* host or device memory; copied at add time          */
  const int8_t *bias;             /* may be NULL (int32 words for LINEAR_OUT_32)        */
  const void *k, *lambda;         /* ch_out values of the network's batch-norm width    */
} pulpnn_layer_desc_t;

pulpnn_net_t *pulpnn_net_create(int bn_bits, int max_batch);
int  pulpnn_net_add_layer(pulpnn_net_t *net, const pulpnn_layer_desc_t *desc);
/* Freezes the layer list and allocates the activation buffers. micro_batch = 0
 * lets the library choose how many images travel through the stack together. */
int  pulpnn_net_finalize(pulpnn_net_t *net, int micro_batch);
/* input: n_images x (first layer's input) bytes; output: n_images x (last
 * layer's output). Either may be host or device memory. Enqueues on the calling
 * thread's stream; synchronises only if a host buffer is involved. */
int  pulpnn_net_run(pulpnn_net_t *net, const uint8_t *input, void *output, int n_images);
/* The same with HOST buffers (pinned memory for real overlap), without waiting: the copies and the
 * kernels of this batch are enqueued and the call returns a ticket (0 or 1; a negative value is
 * minus an error code). pulpnn_net_wait(net, ticket) returns once the batch's results are in
 * `output`. Two batches can be in flight, so in a loop that submits batch i+1 before it waits for
 * batch i the input copy of one batch runs under the compute of the other and the step time is the
 * longer of the two instead of their sum. `input` must stay valid and `output` untouched until the
 * wait; submitting a third batch waits for the first by itself. */
int  pulpnn_net_submit(pulpnn_net_t *net, const uint8_t *input, void *output, int n_images);
int  pulpnn_net_wait(pulpnn_net_t *net, int ticket);
/* Test hook: run the first n_layers layers only and copy that layer's output. */
int  pulpnn_net_run_prefix(pulpnn_net_t *net, const uint8_t *input, void *output, int n_images,
                           int n_layers);
/* Measurement hook: like pulpnn_net_run on device buffers, with a CUDA event recorded on the
 * stream between consecutive layer calls; layer_ms[l] receives the milliseconds layer l took
 * (summed over micro-batches). Synchronises. */
int  pulpnn_net_run_timed(pulpnn_net_t *net, const uint8_t *input, void *output, int n_images,
                          float *layer_ms);
int  pulpnn_net_num_layers(const pulpnn_net_t *net);
size_t pulpnn_net_layer_output_bytes(const pulpnn_net_t *net, int layer);   /* per image */
/* How layer `layer` ran in the most recent run: 0 = a kernel of its own, 1 / 2 = the first /
 * second layer of a pair executed as one fused kernel (PULPNN_OPT_FUSE_DWPW); -1 = no such layer. */
int  pulpnn_net_layer_role(const pulpnn_net_t *net, int layer);
/* The kernel family that ran layer `layer` in the most recent run ("igemm_tc_kernel", ...), for
 * measurement tables; "" before the first run. */
const char *pulpnn_net_layer_kernel(const pulpnn_net_t *net, int layer);
/* Kernel launches the most recent pulpnn_net_run / _run_prefix / _run_timed of this network made
 * (0 before the first run). n_images is ignored. */
unsigned long long pulpnn_net_launches_per_run(const pulpnn_net_t *net, int n_images);
void pulpnn_net_destroy(pulpnn_net_t *net);

#ifdef __cplusplus
}
#endif
#endif /* PULPNN_B200_H */

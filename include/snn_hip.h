/*
 * C ABI of libsnn_hip.so -- the MI355X (gfx950) implementation of portDNN's
 * convolution / depthwise-convolution / pooling hot path.
 *
 * portDNN itself has no C ABI: its boundary is a set of header templates
 * (include/portdnn/<op>/launch.h) over explicitly instantiated launchers that
 * live in libportdnn (src/<op>/launch*.cc).  The entry points below are what a
 * HIP backend for those templates binds, one per (operator, direction, data
 * type); each comment names the reference interface it stands in for.  The
 * C++ drop-in templates in include/portdnn/ are a thin layer over this file.
 *
 * Conventions
 *  - All tensor pointers are DEVICE pointers.  Tensors are NHWC row-major;
 *    dense filters are HWCF [R][S][C][K]; depthwise filters are
 *    [R][S][C][multiplier] and output channel c*multiplier+j.
 *  - `stream` is a hipStream_t passed as void* (NULL = the default stream).
 *    Every call is asynchronous and stream-ordered; no call synchronises.
 *  - The return value is a snn_hip_status.  Values 0..5 are portDNN's
 *    StatusCode enumerators in declaration order
 *    (include/portdnn/status.h:31-44); 6 reports a HIP runtime failure.
 *  - Workspace sizes are counted in ELEMENTS of the data type, as in
 *    include/portdnn/conv2d/workspace_size.h:42-47.
 *  - f16 entry points take IEEE binary16 data and accumulate in fp32.
 */
#ifndef SNN_HIP_H_
#define SNN_HIP_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(_WIN32)
#define SNN_HIP_API
#else
#define SNN_HIP_API __attribute__((visibility("default")))
#endif

typedef enum snn_hip_status {
  SNN_HIP_OK = 0,
  SNN_HIP_INVALID_ALGORITHM = 1,
  SNN_HIP_INDEX_EXCEEDED = 2,
  SNN_HIP_INSUFFICIENT_WORKSPACE = 3,
  SNN_HIP_ALLOCATION_PROBLEM = 4,
  SNN_HIP_INVALID_PARAMETER = 5,
  SNN_HIP_DEVICE_ERROR = 6
} snn_hip_status;

/* sycldnn::conv2d::Algorithm, include/portdnn/conv2d/algorithm.h:30-45 */
typedef enum snn_hip_algorithm {
  SNN_HIP_ALGO_NOT_SUPPORTED = 0,
  SNN_HIP_ALGO_DIRECT = 1,
  SNN_HIP_ALGO_TILED = 2,
  SNN_HIP_ALGO_IM2COL = 3,
  SNN_HIP_ALGO_WINOGRAD = 4,
  SNN_HIP_ALGO_WINOGRAD_LARGE = 5,
  SNN_HIP_ALGO_MATMUL = 6
} snn_hip_algorithm;

/* sycldnn::conv2d::conv_type tags, include/portdnn/conv2d/conv_type.h:35-47 */
typedef enum snn_hip_direction {
  SNN_HIP_FORWARD = 0,
  SNN_HIP_INPUT_BACKPROP = 1,
  SNN_HIP_FILTER_BACKPROP = 2
} snn_hip_direction;

/* POD image of sycldnn::conv2d::Conv2DParams
 * (include/portdnn/conv2d/params.h:32-112), same field order.  The three
 * format fields hold the enumerator values of DataFormat (NHWC = 0, NCHW = 1),
 * FilterFormat (HWCF = 0, FCHW = 1, FHWC = 2) and BatchFormat (STRIDED = 0,
 * INTERLEAVED = 1); only the first of each is accepted. */
typedef struct snn_hip_conv2d_params {
  int channels;
  int features;
  int batch;
  int in_rows;
  int in_cols;
  int window_rows;
  int window_cols;
  int stride_rows;
  int stride_cols;
  int out_rows;
  int out_cols;
  int pad_rows;
  int pad_cols;
  int dilation_rows;
  int dilation_cols;
  int groups;
  int input_format;
  int filter_format;
  int group_format;
} snn_hip_conv2d_params;

/* POD image of sycldnn::depthwise_conv2d::DepthwiseConv2DParams
 * (include/portdnn/depthwise_conv2d/params.h:33-94). */
typedef struct snn_hip_depthwise_params {
  int channels;
  int channel_multiplier;
  int batch;
  int in_rows;
  int in_cols;
  int window_rows;
  int window_cols;
  int stride_rows;
  int stride_cols;
  int out_rows;
  int out_cols;
  int pad_rows;
  int pad_cols;
  int input_format;
  int filter_format;
} snn_hip_depthwise_params;

/* POD image of sycldnn::pooling::PoolingParams
 * (include/portdnn/pooling/params.h:30-73). */
typedef struct snn_hip_pooling_params {
  int in_rows;
  int in_cols;
  int out_rows;
  int out_cols;
  int window_rows;
  int window_cols;
  int stride_rows;
  int stride_cols;
  int batch;
  int channels;
  int pad_rows;
  int pad_cols;
  int input_format;
} snn_hip_pooling_params;

/* sycldnn::pooling operators, include/portdnn/pooling/operators.h:23-42 */
typedef enum snn_hip_pool_op {
  SNN_HIP_POOL_MAX = 0,
  SNN_HIP_POOL_MAX_WITH_NAN = 1,
  SNN_HIP_POOL_AVERAGE = 2
} snn_hip_pool_op;

/* ---- library ------------------------------------------------------------ */

/* Library version, major*10000 + minor*100 + patch. */
SNN_HIP_API int snn_hip_version(void);
/* Static, human-readable name of a status value. */
SNN_HIP_API const char* snn_hip_status_string(int status);
/* Text of the last HIP runtime error seen by the calling thread ("" if none). */
SNN_HIP_API const char* snn_hip_last_error(void);

/* Kernel timing for benchmarks (no counterpart in the reference, whose
 * launches return a cl::sycl::event that carries profiling information).
 * While enabled, every convolution launch brackets its dominant kernel -- the
 * implicit-GEMM or fused Winograd kernel, not the filter preparation or zero
 * fill around it -- with HIP events recorded on the launch stream; depthwise
 * and pooling launches bracket everything they enqueue.
 * snn_hip_kernel_timing_read waits for the recorded events, returns the summed
 * kernel time in milliseconds and the number of kernels, and clears the
 * record.  Launches from several threads may record concurrently (the record
 * is mutex-guarded and stops growing at 65536 kernels until it is read); a
 * read waits for every recorded kernel, so call it from one thread once the
 * timed launches have been enqueued. */
SNN_HIP_API int snn_hip_kernel_timing_enable(int enable);
SNN_HIP_API int snn_hip_kernel_timing_read(double* total_ms, int* kernels);

/* Diagnostics for tests of the tile shapes (no counterpart in portDNN): the
 * tile and the shares of a reduction that the gathering kernel takes for a
 * forward convolution or input gradient behind the Tiled, Im2col and Matmul
 * tags, for aligned operands and a workspace of the recommended size.
 * SNN_HIP_INVALID_ALGORITHM where such a launch runs on another kernel. */
SNN_HIP_API int snn_hip_conv2d_gather_tile(const snn_hip_conv2d_params* params,
                                           int direction, int dtype,
                                           int* pixels, int* features,
                                           int* splits);
/* The tile of the fp32 kernel that takes its operands apart into binary16 values, for
 * a forward convolution or input gradient with this tag; where it answers, such a
 * launch runs there, also one for which the function above has an answer. */
SNN_HIP_API int snn_hip_conv2d_halves_tile(const snn_hip_conv2d_params* params,
                                           int direction, int algorithm,
                                           int* pixels, int* features);
/* The same for the filter gradient: the partial filters that are added up. */
SNN_HIP_API int snn_hip_conv2d_filter_halves_partials(
    const snn_hip_conv2d_params* params, int algorithm, int* partials);
/* The same for the binary16 kernels that keep pixels in LDS: `form` is, for a
 * forward convolution or input gradient, how a work-group of the row-tile kernel
 * holds its input (1: one tile of all channels, 2: two tiles in turn, 3: one tile
 * that is loaded again), and for a filter gradient the work-groups that share a
 * tile of the kernel for 3x3 and 5x5 windows. */
SNN_HIP_API int snn_hip_conv2d_lds_form_f16(const snn_hip_conv2d_params* params,
                                            int direction, int* form);

/* Diagnostics for the stream-ordered temporaries some launches take when the
 * caller passes no workspace (no counterpart in portDNN, whose temporaries
 * come from backend.allocate): bytes currently reserved by, and the high-water
 * mark of bytes in use in, the two pools such temporaries come from on the
 * current device -- the library's own pool and the device's default pool.
 * With reset_high != 0 the high-water marks are cleared after reading, so a
 * caller can bracket a sequence of launches and see whether any of them took
 * a temporary. */
SNN_HIP_API int snn_hip_temporary_memory_stats(
    unsigned long long* reserved_bytes, unsigned long long* used_high_bytes,
    int reset_high);

/* ---- dense convolution ---------------------------------------------------
 * Stand-ins for sycldnn::conv2d::internal::launch_{direct,tiled,matmul,
 * im2col,winograd} reached from sycldnn::conv2d::launch<T, ConvType>
 * (include/portdnn/conv2d/launch.h:59-118 via
 * include/portdnn/internal/conv2d/launch.h:99-207): validate the parameters,
 * check that `algorithm` supports them (SNN_HIP_INVALID_ALGORITHM otherwise,
 * as internal/conv2d/launch.h:127-129,191-197) and enqueue the kernels.
 *
 * forward:         input  [N,H,W,C]    filter [R,S,C,K]    output [N,OH,OW,K]
 * input_backprop:  input = dY [N,OH,OW,K], filter [R,S,C,K], output = dX [N,H,W,C]
 * filter_backprop: input = X [N,H,W,C], filter = dY [N,OH,OW,K], output = dW [R,S,C,K]
 * (operand roles of include/portdnn/conv2d/sizes.h:166-179).
 *
 * `workspace` may be NULL with workspace_elems == 0.  Winograd then returns
 * SNN_HIP_INSUFFICIENT_WORKSPACE (internal/conv2d/winograd/launch.h:271-286);
 * the other algorithms need no caller scratch. */
SNN_HIP_API int snn_hip_conv2d_forward_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_conv2d_params* params, int algorithm, float* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_conv2d_input_backprop_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_conv2d_params* params, int algorithm, float* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_conv2d_filter_backprop_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_conv2d_params* params, int algorithm, float* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_conv2d_forward_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_conv2d_params* params, int algorithm, void* workspace,
    size_t workspace_elems, void* stream);
/* The two gradients in half precision (fp32 accumulation), the reference's
 * launch<half, conv_type::InputBackprop / FilterBackprop>.  Forward
 * convolutions and input gradients of every shape run on binary16 matrix
 * instructions (short ones on fp32 matrix instructions fed binary16 operands,
 * or one lane per output), filter gradients on binary16 ones but for layers of
 * few channels outside the kernels for those, which run in fp32 on widened
 * copies.  No half-precision launch requires a workspace; one of the size
 * snn_hip_conv2d_workspace_size_for reports saves a stream-ordered
 * temporary. */
SNN_HIP_API int snn_hip_conv2d_input_backprop_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_conv2d_params* params, int algorithm, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_conv2d_filter_backprop_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_conv2d_params* params, int algorithm, void* workspace,
    size_t workspace_elems, void* stream);

/* Run-to-run reproducibility.  The reference's kernels add every output's
 * terms in one fixed order, so its results repeat bit for bit.  The entry
 * points above do not always: where a launch would otherwise fill only part
 * of the GPU they split a reduction across work-groups whose partial sums
 * meet through float atomics -- the implicit-GEMM filter gradient (Im2col /
 * Tiled / Direct-fallback tags) always, except for the 7x7 stride-2
 * three-channel stem from 224 output rows over the batch upwards and for
 * every other layer with at least 32 channels, or with window size x channels
 * above 192, or with a feature count that is not a multiple of 4 (16-byte
 * aligned operands, at least 256 output pixels), whose partial filters are
 * summed in a fixed order; forward and input gradients of small
 * problems (fewer than ~640 64x64 output tiles, unless one of the kernels
 * that sum their parts in a fixed order takes the launch: stride-1 layers
 * with channels in multiples of 128, forward problems of fewer than 128
 * tiles) and the fused Winograd
 * kernel below 128 work units -- and the order of those additions, hence the
 * last bits of the result, can change between runs.  The Winograd filter
 * gradient and every launch without such a split are reproducible.
 *
 * snn_hip_conv2d_deterministic_f32 is the same operation as the three fp32
 * entry points (`direction` is a snn_hip_direction) with a fixed order of
 * additions: no reduction splits (small problems run on fewer work-groups),
 * and a filter gradient outside the Winograd algorithm runs on the direct
 * kernel, one lane per filter element (the layers named above keep their
 * kernel).  Two calls with the same arguments
 * return bit-identical results.  Workspace sizes are those of
 * snn_hip_conv2d_workspace_size. */
SNN_HIP_API int snn_hip_conv2d_deterministic_f32(
    int direction, const float* input, const float* filter, float* output,
    const snn_hip_conv2d_params* params, int algorithm, float* workspace,
    size_t workspace_elems, void* stream);

/* A launch in two calls, for callers that run many launches with one filter
 * (inference).  No counterpart in portDNN, whose Winograd launch transforms
 * the filter every time (internal/conv2d/winograd/launch.h:212-235).
 *
 * snn_hip_conv2d_prepare_filter_f32 writes into `workspace` whatever a launch
 * with these parameters, direction and algorithm derives from the filter
 * alone -- today, for forward convolutions and input gradients behind the
 * Winograd tags, the fused kernels' transformed filter or the filter as two
 * binary16 values per weight, whichever kernel the sizes choose; for every other
 * path it does nothing and returns SNN_HIP_OK.  snn_hip_conv2d_prepared_f32 is then the same operation as the
 * three fp32 entry points, except that it trusts those contents instead of
 * recomputing them: the caller guarantees that `workspace` (same pointer,
 * same size) still holds what a prepare call with the same filter values,
 * parameters, direction and algorithm wrote, and that nothing else wrote to
 * its first 16 * C * K elements since.  Where something was prepared the
 * launch only reads the workspace, whichever kernel it takes, so that launches
 * on several streams may share one.  The one-call entry points never trust a
 * workspace: they always transform the filter they are given. */
SNN_HIP_API int snn_hip_conv2d_prepare_filter_f32(
    int direction, const float* filter, const snn_hip_conv2d_params* params,
    int algorithm, float* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_conv2d_prepared_f32(
    int direction, const float* input, const float* filter, float* output,
    const snn_hip_conv2d_params* params, int algorithm, float* workspace,
    size_t workspace_elems, void* stream);

/* sycldnn::conv2d::query_workspace_size<ConvType>(params, selector)
 * (include/portdnn/conv2d/workspace_size.h:158-163) for an already selected
 * algorithm.  Sizes in elements. */
SNN_HIP_API int snn_hip_conv2d_workspace_size(
    const snn_hip_conv2d_params* params, int direction, int algorithm,
    size_t* required_elems, size_t* recommended_elems);

/* The same for a given element type (a snn_hip_dtype), in elements of that
 * type.  portDNN's query does not know the element type
 * (workspace_size.h:158-163 takes only the parameters and the selector); the
 * half-precision kernels here are different kernels with different needs, so
 * a caller that sizes its scratch from the fp32 answer would allocate the
 * F(2x2,3x3) transform buffers for a launch that uses a filter-sized block.
 * For SNN_HIP_DTYPE_F16 `required` is always 0 (a launch without scratch
 * takes a stream-ordered temporary) and `recommended` is what the launch
 * uses.  SNN_HIP_DTYPE_F32 answers as snn_hip_conv2d_workspace_size. */
typedef enum snn_hip_dtype {
  SNN_HIP_DTYPE_F32 = 0,
  SNN_HIP_DTYPE_F16 = 1,
  /* bfloat16: the operators of a residual block over sequences only */
  SNN_HIP_DTYPE_BF16 = 2
} snn_hip_dtype;
SNN_HIP_API int snn_hip_conv2d_workspace_size_for(
    const snn_hip_conv2d_params* params, int direction, int algorithm,
    int dtype, size_t* required_elems, size_t* recommended_elems);

/* Does `algorithm` support these parameters in this direction?  Mirrors the
 * concrete selectors (include/portdnn/conv2d/selector/{tiled,winograd,matmul}_
 * selector.h, constant_selector.h): returns `algorithm` if it does, else
 * SNN_HIP_ALGO_NOT_SUPPORTED. */
SNN_HIP_API int snn_hip_conv2d_algorithm_supports(
    const snn_hip_conv2d_params* params, int direction, int algorithm);

/* The algorithm sycldnn::conv2d::get_default_selector(device) would pick on
 * this device (src/conv2d/selector/default_selector.cc:257-286), tuned for
 * MI355X. */
SNN_HIP_API int snn_hip_conv2d_default_algorithm(
    const snn_hip_conv2d_params* params, int direction);
/* The same for a given element type: half precision has no Winograd kernels,
 * so its 3x3 layers get the Tiled (forward) / Im2col tag, whose kernels and
 * workspace snn_hip_conv2d_workspace_size_for describes. */
SNN_HIP_API int snn_hip_conv2d_default_algorithm_for(
    const snn_hip_conv2d_params* params, int direction, int dtype);

/* ---- depthwise convolution -----------------------------------------------
 * Stand-ins for sycldnn::depthwise_conv2d::internal::launch<ConvType>
 * (src/depthwise_conv2d/launch.cc:100-121) reached from
 * sycldnn::depthwise_conv2d::launch (include/portdnn/depthwise_conv2d/
 * launch.h:54-91).  Operand roles as for the dense convolution with
 * K = C * multiplier. */
SNN_HIP_API int snn_hip_depthwise_conv2d_forward_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_depthwise_params* params, void* stream);
SNN_HIP_API int snn_hip_depthwise_conv2d_input_backprop_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_depthwise_params* params, void* stream);
SNN_HIP_API int snn_hip_depthwise_conv2d_filter_backprop_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_depthwise_params* params, void* stream);
/* The fp32 filter gradient for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  No counterpart in the reference.  Same operands and result as
 * snn_hip_depthwise_conv2d_filter_backprop_f32, whose large-input path keeps
 * the work-groups' partial filters in a stream-ordered temporary; here they
 * live in a 9 MiB device array inside the library (held by every GPU the
 * library runs on until the process ends), sized for the largest plan that
 * path makes, so no hipMalloc / hipFree in any form is called.  A shape whose
 * partial filters would not fit is rejected with SNN_HIP_INVALID_PARAMETER
 * and a message in snn_hip_last_error().  All calls on one GPU share that
 * array: calls that overlap on one GPU (different streams or threads) race;
 * stream-ordered calls are safe.  The stream's device must be current.  The
 * first call on each device looks the array's address up
 * (hipGetSymbolAddress, which may load the library's device code): make one
 * call per device before a stream capture begins; later calls only enqueue
 * kernels. */
SNN_HIP_API int snn_hip_depthwise_conv2d_filter_backprop_noalloc_f32(
    const float* input, const float* filter, float* output,
    const snn_hip_depthwise_params* params, void* stream);
SNN_HIP_API int snn_hip_depthwise_conv2d_forward_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_depthwise_params* params, void* stream);
SNN_HIP_API int snn_hip_depthwise_conv2d_input_backprop_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_depthwise_params* params, void* stream);
SNN_HIP_API int snn_hip_depthwise_conv2d_filter_backprop_f16(
    const void* input, const void* filter, void* output,
    const snn_hip_depthwise_params* params, void* stream);

/* ---- pooling -------------------------------------------------------------
 * Stand-ins for sycldnn::pooling::internal::launch_pooling
 * (src/pooling/launch_pooling.cc:146-165) reached from
 * sycldnn::pooling::launch<T, PoolType, Direction>
 * (include/portdnn/pooling/launch.h:112-128 forward, :153-172 max gradient).
 * `op` is a snn_hip_pool_op. */
SNN_HIP_API int snn_hip_pooling_forward_f32(
    const float* input, float* output, const snn_hip_pooling_params* params,
    int op, void* stream);
SNN_HIP_API int snn_hip_pooling_forward_f16(
    const void* input, void* output, const snn_hip_pooling_params* params,
    int op, void* stream);
/* Max / MaxWithNan gradient: input_data and output_data are the forward
 * tensors, input_backprop is dY [N,OH,OW,C], output_backprop is dX [N,H,W,C]. */
SNN_HIP_API int snn_hip_pooling_max_grad_f32(
    const float* input_data, const float* output_data,
    const float* input_backprop, float* output_backprop,
    const snn_hip_pooling_params* params, int op, void* stream);
/* Average gradient: input_backprop dY [N,OH,OW,C] -> output_backprop dX. */
SNN_HIP_API int snn_hip_pooling_avg_grad_f32(
    const float* input_backprop, float* output_backprop,
    const snn_hip_pooling_params* params, void* stream);
/* The two gradients on half-precision tensors (same operands). */
SNN_HIP_API int snn_hip_pooling_max_grad_f16(
    const void* input_data, const void* output_data,
    const void* input_backprop, void* output_backprop,
    const snn_hip_pooling_params* params, int op, void* stream);
SNN_HIP_API int snn_hip_pooling_avg_grad_f16(
    const void* input_backprop, void* output_backprop,
    const snn_hip_pooling_params* params, void* stream);

/* ---- matmul ----------------------------------------------------------------
 * Stand-in for sycldnn::matmul::internal::launch (src/matmul/launch.cc) as the
 * backend's matmul / batch_matmul members call it
 * (include/portdnn/backend/snn_usm_matmul_provider.h:206-231): row-major
 * C[b] = op(A[b]) * op(B[b]) + beta * C[b], op(A) m x k, op(B) k x n. */
SNN_HIP_API int snn_hip_matmul_f32(const float* lhs, const float* rhs,
                                   float* output, int batches, int m, int k,
                                   int n, int transpose_lhs, int transpose_rhs,
                                   float beta, void* stream);
/* The same on half-precision matrices (products and sums in fp32). */
SNN_HIP_API int snn_hip_matmul_f16(const void* lhs, const void* rhs,
                                   void* output, int batches, int m, int k,
                                   int n, int transpose_lhs, int transpose_rhs,
                                   float beta, void* stream);

/* ---- convolution with bias and activation ---------------------------------
 * No single counterpart in the reference, which runs three launches for this
 * (conv2d::launch, binaryop::launch<Add> with the bias as a [features]
 * operand, pointwise::launch<Relu, Forward>; e.g. the layers of
 * tools/layer.h).  Here the bias add and the activation are folded into the
 * convolution's output stage wherever the chosen kernel writes each output
 * once, and run as one in-place pass otherwise; the result equals the three
 * launches.  `bias` holds one value per feature or is NULL; `activation` is a
 * snn_hip_activation.  Everything else as snn_hip_conv2d_forward_f32. */
typedef enum snn_hip_activation {
  SNN_HIP_ACTIVATION_NONE = 0,
  SNN_HIP_ACTIVATION_RELU = 1,
  /* snn_hip_matmul_bias_act_* only: z Phi(z), its approximation through
   * tanh(sqrt(2 / pi) (z + 0.044715 z^3)), and z sigmoid(z). */
  SNN_HIP_ACTIVATION_GELU = 2,
  SNN_HIP_ACTIVATION_GELU_TANH = 3,
  SNN_HIP_ACTIVATION_SILU = 4
} snn_hip_activation;
SNN_HIP_API int snn_hip_conv2d_forward_bias_act_f32(
    const float* input, const float* filter, const float* bias, float* output,
    const snn_hip_conv2d_params* params, int algorithm, int activation,
    float* workspace, size_t workspace_elems, void* stream);

/* ---- alpha / beta blend ----------------------------------------------------
 * data[i] = alpha * data[i] + beta * prior[i] over n_items elements: the
 * scaling step of the cuDNN-style layer (ScalingParams::applyScaling,
 * include/portdnn/compat/scaling.hpp:150-262, which composes binaryop
 * launches for it).  `prior` may be NULL when beta is 0; a zero alpha drops
 * the data term outright. */
SNN_HIP_API int snn_hip_scale_blend_f32(float* data, const float* prior,
                                        float alpha, float beta,
                                        size_t n_items, void* stream);

/* ---- pointwise -------------------------------------------------------------
 * Stand-ins for sycldnn::pointwise::internal::launch_pointwise
 * (src/pointwise/launch_pointwise_forward.cc, launch_pointwise_grad.cc)
 * reached from sycldnn::pointwise::launch<T, Op, Direction>
 * (include/portdnn/pointwise/launch.h:73-100 forward, :120-150 gradient).
 * `op` is a snn_hip_pointwise_op; n_items must be positive
 * (include/portdnn/internal/pointwise/launch_internal.h:69). */
typedef enum snn_hip_pointwise_op {
  SNN_HIP_POINTWISE_RELU = 0,
  SNN_HIP_POINTWISE_TANH = 1,
  SNN_HIP_POINTWISE_EXP = 2,
  SNN_HIP_POINTWISE_LOG = 3,
  SNN_HIP_POINTWISE_FLOOR = 4,
  SNN_HIP_POINTWISE_SQRT = 5
} snn_hip_pointwise_op;
SNN_HIP_API int snn_hip_pointwise_forward_f32(const float* input, float* output,
                                              size_t n_items, int op,
                                              void* stream);
SNN_HIP_API int snn_hip_pointwise_forward_f16(const void* input, void* output,
                                              size_t n_items, int op,
                                              void* stream);
/* Gradient: input_forward is what the reference's operators call `val` (the
 * forward OUTPUT for relu, tanh, exp and sqrt, the forward INPUT for log;
 * src/pointwise/kernels.h:53-57, :75-77, :100-102, :122-124, :158-160),
 * input_backprop the incoming error.  Floor has no gradient. */
SNN_HIP_API int snn_hip_pointwise_grad_f32(const float* input_forward,
                                           const float* input_backprop,
                                           float* output_backprop,
                                           size_t n_items, int op,
                                           void* stream);
SNN_HIP_API int snn_hip_pointwise_grad_f16(const void* input_forward,
                                           const void* input_backprop,
                                           void* output_backprop,
                                           size_t n_items, int op,
                                           void* stream);

/* ---- binaryop --------------------------------------------------------------
 * Stand-ins for sycldnn::binaryop::internal::launch_binaryop
 * (src/binaryop/launch_binaryop.cc) reached from
 * sycldnn::binaryop::launch<T, Op>
 * (include/portdnn/binaryop/launch.h:61-85).  The dimension lists are
 * BinaryParams::lhs_dims / rhs_dims (include/portdnn/binaryop/params.h:37-46):
 * at most four each (none = scalar), right-aligned, a dimension of 1
 * broadcasts; shapes that do not broadcast return
 * SNN_HIP_INVALID_PARAMETER
 * (include/portdnn/internal/binaryop/launch.h:40-62). */
typedef enum snn_hip_binary_op {
  SNN_HIP_BINARY_ADD = 0,
  SNN_HIP_BINARY_SUB = 1,
  SNN_HIP_BINARY_MUL = 2,
  SNN_HIP_BINARY_DIV = 3
} snn_hip_binary_op;
SNN_HIP_API int snn_hip_binaryop_f32(const float* lhs, const float* rhs,
                                     float* output, const int* lhs_dims,
                                     int n_lhs_dims, const int* rhs_dims,
                                     int n_rhs_dims, int op, void* stream);
SNN_HIP_API int snn_hip_binaryop_f16(const void* lhs, const void* rhs,
                                     void* output, const int* lhs_dims,
                                     int n_lhs_dims, const int* rhs_dims,
                                     int n_rhs_dims, int op, void* stream);

/* ---- a residual block over sequences ---------------------------------------
 * Operators of language models that portDNN has no counterpart of: a matrix
 * product with its epilogue, the norms around a block and a gated linear
 * recurrence.  Tensors are row-major with the channels innermost, so that a
 * [batch, steps, channels] tensor is the NHWC tensor of one row of `steps`
 * columns.  Data types: float, IEEE binary16 (_f16) and bfloat16 (_bf16);
 * sums, statistics and states are fp32, and an output is rounded to its type
 * once.  A stride is the number of elements from one row to the next, at least
 * the row's length; 0 stands for rows that follow one another. */

/* output = act(op(lhs) op(rhs) + bias) + residual.
 *
 * op(lhs) is m x k: stored m x k, or k x m when transpose_lhs; op(rhs) is
 * k x n: stored k x n, or n x k when transpose_rhs.  bias holds n values,
 * residual and output are m x n.  bias, residual and pre_activation may be
 * NULL; pre_activation, m x n without a stride, receives the value in front of
 * the activation, which the gradient takes.  residual may be output (the sum
 * in place); no other operand may overlap an output.
 *
 * Every dimension is positive and every row shorter than 2^30 bytes; tensors
 * may be of any size beyond that, as far as a grid holds the output's tiles
 * (SNN_HIP_INDEX_EXCEEDED; from 2^35 values on).  A workspace of the recommended size lets
 * products with few output tiles share their reduction between work-groups (the
 * parts are added in a fixed order: two calls with the same arguments, workspace
 * included, return the same bits) and holds copies of operands whose rows do not
 * start at multiples of 16 bytes; without it products run on fewer work-groups,
 * or on slower kernels. */
typedef struct snn_hip_matmul_bias_act_params {
  int m;
  int k;
  int n;
  int transpose_lhs;
  int transpose_rhs;
  int activation; /* a snn_hip_activation */
  int lhs_stride;
  int rhs_stride;
  int residual_stride;
  int output_stride;
} snn_hip_matmul_bias_act_params;
SNN_HIP_API int snn_hip_matmul_bias_act_f32(
    const void* lhs, const void* rhs, const void* bias, const void* residual,
    void* output, void* pre_activation,
    const snn_hip_matmul_bias_act_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_matmul_bias_act_f16(
    const void* lhs, const void* rhs, const void* bias, const void* residual,
    void* output, void* pre_activation,
    const snn_hip_matmul_bias_act_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_matmul_bias_act_bf16(
    const void* lhs, const void* rhs, const void* bias, const void* residual,
    void* output, void* pre_activation,
    const snn_hip_matmul_bias_act_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* The gradients.  grad_output is m x n with the stride output_stride (it is
 * the residual's gradient as it stands), pre_activation what the forward call
 * wrote (not read where activation is none).  grad_lhs and grad_rhs are stored
 * as lhs and rhs are, transposed or not, without a stride; grad_bias holds n
 * values.  Any of the three may be NULL and is then not computed; lhs is needed
 * for grad_rhs and rhs for grad_lhs only.  grad_bias and, where there is an
 * activation, the products (which need the gradient with respect to
 * pre_activation, rounded to the data type: in binary16 it is infinite beyond
 * 65504) take workspace: SNN_HIP_INSUFFICIENT_WORKSPACE without the required
 * size. */
SNN_HIP_API int snn_hip_matmul_bias_act_grad_f32(
    const void* grad_output, const void* lhs, const void* rhs,
    const void* pre_activation, void* grad_lhs, void* grad_rhs,
    void* grad_bias, const snn_hip_matmul_bias_act_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_matmul_bias_act_grad_f16(
    const void* grad_output, const void* lhs, const void* rhs,
    const void* pre_activation, void* grad_lhs, void* grad_rhs,
    void* grad_bias, const snn_hip_matmul_bias_act_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_matmul_bias_act_grad_bf16(
    const void* grad_output, const void* lhs, const void* rhs,
    const void* pre_activation, void* grad_lhs, void* grad_rhs,
    void* grad_bias, const snn_hip_matmul_bias_act_params* params,
    void* workspace, size_t workspace_elems, void* stream);
/* Workspace of the forward call (grad == 0) or of the gradients, in elements
 * of `dtype`; the pointer is aligned to 16 bytes, as all workspaces of this
 * section are. */
SNN_HIP_API int snn_hip_matmul_bias_act_workspace_size(
    const snn_hip_matmul_bias_act_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems);
/* Diagnostics for tests of the kernels: what a product runs on, given a workspace
 * of `workspace_elems`, and operands that start at multiples of 16 bytes or do not.
 * `product` is 0 for the forward call, 1 and 2 for grad_lhs and grad_rhs of a call
 * for all three gradients.  The result's rows are the first operand's. */
typedef struct snn_hip_matmul_bias_act_plan {
  int tile_rows;
  int tile_cols;
  int shared;       /* 1: a tile's reduction is shared by the work-group's waves */
  int any_address;  /* 1: operands by way of registers, 0: straight to LDS */
  int pair;         /* 1: two work-groups to a CU */
  int first_inner;  /* 1: the reduction is contiguous in the first operand */
  int second_inner; /* ... and in the second */
  int first_copied; /* 1: copied to aligned rows first */
  int second_copied;
  int shares;       /* of the reduction, each by a work-group of its own */
} snn_hip_matmul_bias_act_plan;
SNN_HIP_API int snn_hip_matmul_bias_act_planned(
    const snn_hip_matmul_bias_act_params* params, int product, int dtype,
    int aligned, size_t workspace_elems, snn_hip_matmul_bias_act_plan* plan);

/* The norms before and after a block, with its gate and residual scale, in
 * one pass over the rows:
 *
 *   n = post_norm(x) * post_weight + post_bias     the block's output
 *   sum = residual + scale * gate * n              the residual stream
 *   normed = pre_norm(sum) * pre_weight + pre_bias the next block's input
 *
 * x, residual, sum and normed are rows x channels; scale and the norms'
 * weights and biases hold one value per channel; the gate has one row for
 * `gate_rows` consecutive rows of x (1: one for each) and enters as it is,
 * through a sigmoid, or as gate * sigmoid(gate).  A norm divides by
 * sqrt(mean(v^2) + epsilon) (RMS) or takes the mean out first (LAYER).
 * residual, gate, scale, the weights and biases, sum, normed and stats may be
 * NULL; weights and biases of an absent norm have to be, normed has to be
 * where there is no pre_norm, and sum or normed has to be there.  `gate` and
 * the operand are both there or both not.  stats (rows x 4 floats) receives
 * mean and reciprocal deviation of the two norms, zeros for what a row has
 * not, for the gradients.  sum may be x or residual (with the stride of x
 * that sum has); no other output may overlap an input.  At most 16384
 * channels. */
typedef enum snn_hip_norm {
  SNN_HIP_NORM_NONE = 0,
  SNN_HIP_NORM_RMS = 1,
  SNN_HIP_NORM_LAYER = 2
} snn_hip_norm;
typedef enum snn_hip_gate {
  SNN_HIP_GATE_NONE = 0,
  SNN_HIP_GATE_VALUE = 1,
  SNN_HIP_GATE_SIGMOID = 2,
  SNN_HIP_GATE_SILU = 3
} snn_hip_gate;
typedef struct snn_hip_residual_norm_params {
  int rows;
  int channels;
  int post_norm; /* a snn_hip_norm */
  int pre_norm;  /* a snn_hip_norm */
  int gate;      /* a snn_hip_gate */
  int gate_rows;
  int x_stride;    /* of x */
  int gate_stride; /* of the gate */
  float epsilon;
} snn_hip_residual_norm_params;
typedef struct snn_hip_residual_norm_tensors {
  const void* x;
  const void* residual;
  const void* gate;
  const void* scale;
  const void* post_weight;
  const void* post_bias;
  const void* pre_weight;
  const void* pre_bias;
  void* sum;
  void* normed;
  float* stats;
} snn_hip_residual_norm_tensors;
SNN_HIP_API int snn_hip_residual_norm_f32(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_params* params, void* stream);
SNN_HIP_API int snn_hip_residual_norm_f16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_params* params, void* stream);
SNN_HIP_API int snn_hip_residual_norm_bf16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_params* params, void* stream);
/* The gradients.  `tensors` holds the forward call's operands and its sum and
 * stats (residual and normed are not read, sum is read where there is a
 * pre_norm, stats where there is any norm).  grad_sum and grad_normed are the
 * gradients of the two outputs (either may be NULL; grad_normed has to be
 * where there is no pre_norm); the others are outputs without strides, NULL
 * where they are not wanted.  The weights', biases', scale's and a shared
 * gate's gradients are sums over rows, added in a fixed order; their partial
 * sums take the required workspace. */
typedef struct snn_hip_residual_norm_gradients {
  const void* grad_sum;
  const void* grad_normed;
  void* grad_x;
  void* grad_residual;
  void* grad_gate;
  void* grad_scale;
  void* grad_post_weight;
  void* grad_post_bias;
  void* grad_pre_weight;
  void* grad_pre_bias;
} snn_hip_residual_norm_gradients;
SNN_HIP_API int snn_hip_residual_norm_grad_f32(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_residual_norm_grad_f16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_residual_norm_grad_bf16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* Workspace of the gradients in elements of `dtype`, enough for all of them;
 * the sums over rows need the required size, the others none. */
SNN_HIP_API int snn_hip_residual_norm_grad_workspace_size(
    const snn_hip_residual_norm_params* params, int dtype,
    size_t* required_elems, size_t* recommended_elems);

/* A gated linear recurrence over the steps of a sequence, channel by channel:
 *
 *   a_t = sigmoid(forget_t)
 *   b_t = w_t x_t,  w_t = sigmoid(input_gate_t), or 1 - a_t without that gate
 *   h_t = a_t h_{t-1} + b_t
 *
 * x, forget and input_gate are [batch][steps][channels] with row_stride
 * elements from step to step (steps * row_stride from sequence to sequence),
 * so that they may be slices of one projection's output; h is
 * [batch][steps][channels] without a stride.  initial_state and final_state
 * are [batch][channels] floats (NULL: zero, not wanted) and may be one buffer:
 * a single token is a call with one step that updates the state in place.
 * resets ([batch][steps] bytes, NULL: none): where it is not zero a_t h_{t-1}
 * is left out, whatever it is, so that a sequence may hold several documents.
 * lengths ([batch] ints, NULL: all steps; clamped to 0 ... steps): steps from
 * there on are not read, their h is zero, and final_state is the state behind
 * the last step that counts (the initial state for a length of zero).
 *
 * Long sequences are divided into pieces that run beside one another, given a
 * workspace of the recommended size; without one a sequence is one piece.  The
 * order of operations is fixed by the sizes and the workspace. */
typedef struct snn_hip_linear_recurrence_params {
  int batch;
  int steps;
  int channels;
  int row_stride;      /* of x, forget and input_gate */
  int grad_row_stride; /* of their gradients */
} snn_hip_linear_recurrence_params;
SNN_HIP_API int snn_hip_linear_recurrence_f32(
    const void* x, const void* forget, const void* input_gate,
    const unsigned char* resets, const int* lengths,
    const float* initial_state, void* h, float* final_state,
    const snn_hip_linear_recurrence_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_recurrence_f16(
    const void* x, const void* forget, const void* input_gate,
    const unsigned char* resets, const int* lengths,
    const float* initial_state, void* h, float* final_state,
    const snn_hip_linear_recurrence_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_recurrence_bf16(
    const void* x, const void* forget, const void* input_gate,
    const unsigned char* resets, const int* lengths,
    const float* initial_state, void* h, float* final_state,
    const snn_hip_linear_recurrence_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* The gradients: `h` is what the forward call wrote, grad_final_state may be
 * NULL.  grad_x, grad_forget and grad_input_gate (which is there exactly where
 * input_gate is) have grad_row_stride and are zero from a sequence's length
 * on; grad_initial_state may be NULL or grad_final_state. */
SNN_HIP_API int snn_hip_linear_recurrence_grad_f32(
    const void* grad_h, const float* grad_final_state, const void* x,
    const void* forget, const void* input_gate, const unsigned char* resets,
    const int* lengths, const float* initial_state, const void* h,
    void* grad_x, void* grad_forget, void* grad_input_gate,
    float* grad_initial_state, const snn_hip_linear_recurrence_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_recurrence_grad_f16(
    const void* grad_h, const float* grad_final_state, const void* x,
    const void* forget, const void* input_gate, const unsigned char* resets,
    const int* lengths, const float* initial_state, const void* h,
    void* grad_x, void* grad_forget, void* grad_input_gate,
    float* grad_initial_state, const snn_hip_linear_recurrence_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_recurrence_grad_bf16(
    const void* grad_h, const float* grad_final_state, const void* x,
    const void* forget, const void* input_gate, const unsigned char* resets,
    const int* lengths, const float* initial_state, const void* h,
    void* grad_x, void* grad_forget, void* grad_input_gate,
    float* grad_initial_state, const snn_hip_linear_recurrence_params* params,
    void* workspace, size_t workspace_elems, void* stream);
/* Workspace of either call, in elements of `dtype`; none is required.  Sequences
 * of more than 2^31 - 65 steps or 2^31 - 1025 channels, and more than 2^31 - 1
 * sequences times blocks of 64 channels, are SNN_HIP_INDEX_EXCEEDED here and in
 * the calls. */
SNN_HIP_API int snn_hip_linear_recurrence_workspace_size(
    const snn_hip_linear_recurrence_params* params, int dtype,
    size_t* required_elems, size_t* recommended_elems);

/* ---- a linear-attention block ------------------------------------------------
 * What a block of linear attention takes beside the operators above: a product
 * gated by another, positions by rotation, and the attention itself, a
 * recurrence whose state is a matrix for each head.  Types, strides, rounding
 * and workspaces as above. */

/* output = act(lhs op(gate_weight) + gate_bias) * (lhs op(up_weight) + up_bias):
 * the first half of a gated feed-forward part, both products in one pass over
 * lhs.  (Its second half is a matrix product with a residual.)
 *
 * lhs is m x k; both weights are stored k x n, or n x k when transpose_rhs, with
 * one stride, so that they may be the two halves of one matrix.  The biases hold
 * n values; either may be NULL.  gate and up, m x n without a stride, both NULL or
 * both there, receive the two factors' values in front of the activation, which
 * the gradients take.  No operand may overlap an output.  Sizes, workspace and
 * order of sums as in snn_hip_matmul_bias_act. */
typedef struct snn_hip_gated_matmul_params {
  int m;
  int k;
  int n;
  int transpose_rhs;
  int activation; /* a snn_hip_activation */
  int lhs_stride;
  int rhs_stride;    /* of both weights */
  int output_stride; /* of output and grad_output */
} snn_hip_gated_matmul_params;
SNN_HIP_API int snn_hip_gated_matmul_f32(
    const void* lhs, const void* gate_weight, const void* up_weight,
    const void* gate_bias, const void* up_bias, void* output, void* gate,
    void* up, const snn_hip_gated_matmul_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_gated_matmul_f16(
    const void* lhs, const void* gate_weight, const void* up_weight,
    const void* gate_bias, const void* up_bias, void* output, void* gate,
    void* up, const snn_hip_gated_matmul_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_gated_matmul_bf16(
    const void* lhs, const void* gate_weight, const void* up_weight,
    const void* gate_bias, const void* up_bias, void* output, void* gate,
    void* up, const snn_hip_gated_matmul_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* The gradients; gate and up are what the forward call wrote.  grad_lhs and the
 * weights' gradients are stored as those are, without a stride; each of the five
 * may be NULL and is then not computed.  lhs is needed for the weights' gradients
 * and both weights for grad_lhs only.  The gradients of the two factors, rounded to
 * the data type (in binary16: infinite beyond 65504, in steps of 2^-24 below 2^-14),
 * and the biases' sums take workspace:
 * SNN_HIP_INSUFFICIENT_WORKSPACE without the required size. */
SNN_HIP_API int snn_hip_gated_matmul_grad_f32(
    const void* grad_output, const void* lhs, const void* gate_weight,
    const void* up_weight, const void* gate, const void* up, void* grad_lhs,
    void* grad_gate_weight, void* grad_up_weight, void* grad_gate_bias,
    void* grad_up_bias, const snn_hip_gated_matmul_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_gated_matmul_grad_f16(
    const void* grad_output, const void* lhs, const void* gate_weight,
    const void* up_weight, const void* gate, const void* up, void* grad_lhs,
    void* grad_gate_weight, void* grad_up_weight, void* grad_gate_bias,
    void* grad_up_bias, const snn_hip_gated_matmul_params* params,
    void* workspace, size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_gated_matmul_grad_bf16(
    const void* grad_output, const void* lhs, const void* gate_weight,
    const void* up_weight, const void* gate, const void* up, void* grad_lhs,
    void* grad_gate_weight, void* grad_up_weight, void* grad_gate_bias,
    void* grad_up_bias, const snn_hip_gated_matmul_params* params,
    void* workspace, size_t workspace_elems, void* stream);
/* Workspace of the forward call (grad == 0) or of the gradients, in elements of
 * `dtype`. */
SNN_HIP_API int snn_hip_gated_matmul_workspace_size(
    const snn_hip_gated_matmul_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems);
/* Diagnostics for tests of the kernels, as snn_hip_matmul_bias_act_planned: `product`
 * is 0 for the forward call, 1 for grad_lhs and 2 for a weight's gradient of a call for
 * all five gradients.  tile_cols are those of both weights together (0), and both
 * weights or both factors are copied or neither is. */
SNN_HIP_API int snn_hip_gated_matmul_planned(
    const snn_hip_gated_matmul_params* params, int product, int dtype,
    int aligned, size_t workspace_elems, snn_hip_matmul_bias_act_plan* plan);

/* Positions by rotation.  Of each head's `channels` the first `turned` form pairs
 * (a, b), channel i with i + turned / 2 (HALVES) or 2 i with 2 i + 1 (PAIRS), and
 * pair i of a token at position p becomes
 *
 *   magnitude (a cos w - b sin w),  magnitude (a sin w + b cos w)
 *
 * with w = 2 pi p frequencies[i], or -w where `inverse` is set: the gradient of
 * the forward call is the inverse call on the output's gradient.  The other
 * channels are copied as they are.  Angles are reduced in 64 bits, so that far
 * positions lose nothing.
 *
 * input is [batch][steps][heads][channels] with row_stride elements from step to
 * step (steps * row_stride from sequence to sequence), output the same with
 * output_row_stride, so that both may be slices of a projection's rows; output may
 * be input with the same stride (in place), otherwise they may not overlap.
 * `positions` is NULL where params->positions is NONE (a token's position is its
 * step), [batch] ints for FIRST (the position of step 0, the others follow) or
 * [batch][steps] for EACH.  2^32 or more lanes, tokens times groups of 16 bytes of a
 * head, are SNN_HIP_INDEX_EXCEEDED. */
typedef enum snn_hip_rotary_layout {
  SNN_HIP_ROTARY_HALVES = 0,
  SNN_HIP_ROTARY_PAIRS = 1
} snn_hip_rotary_layout;
typedef enum snn_hip_rotary_positions {
  SNN_HIP_ROTARY_POSITIONS_NONE = 0,
  SNN_HIP_ROTARY_POSITIONS_FIRST = 1,
  SNN_HIP_ROTARY_POSITIONS_EACH = 2
} snn_hip_rotary_positions;
typedef struct snn_hip_rotary_params {
  int batch;
  int steps;
  int heads;
  int channels; /* of a head */
  int turned;   /* even, 2 ... channels */
  int layout;   /* a snn_hip_rotary_layout */
  int positions; /* a snn_hip_rotary_positions */
  int inverse;
  int row_stride;
  int output_row_stride;
  float magnitude;
} snn_hip_rotary_params;
SNN_HIP_API int snn_hip_rotary_f32(const void* input, const double* frequencies,
                                   const int* positions, void* output,
                                   const snn_hip_rotary_params* params,
                                   void* stream);
SNN_HIP_API int snn_hip_rotary_f16(const void* input, const double* frequencies,
                                   const int* positions, void* output,
                                   const snn_hip_rotary_params* params,
                                   void* stream);
SNN_HIP_API int snn_hip_rotary_bf16(const void* input,
                                    const double* frequencies,
                                    const int* positions, void* output,
                                    const snn_hip_rotary_params* params,
                                    void* stream);
/* The frequencies of turned / 2 pairs, in turns from one position to the next:
 * base^(-2 i / turned) / (2 pi), written to `frequencies` in host memory, which the
 * calls above take from device memory.  For contexts `factor` times the `context`
 * tokens that a model has been trained on:
 *
 *   POSITIONS  every frequency divided by factor;
 *   BASE       the base times factor^(turned / (turned - 2)): the first pair stays,
 *              the last is divided by factor;
 *   BANDS      pairs of at least `high` turns within the context stay, those of
 *              at most `low` are divided by factor, between them the two are
 *              mixed in proportion to the turns.
 *
 * `context`, `low` and `high` are read for BANDS only. */
typedef enum snn_hip_rotary_scaling {
  SNN_HIP_ROTARY_SCALING_NONE = 0,
  SNN_HIP_ROTARY_SCALING_POSITIONS = 1,
  SNN_HIP_ROTARY_SCALING_BASE = 2,
  SNN_HIP_ROTARY_SCALING_BANDS = 3
} snn_hip_rotary_scaling;
SNN_HIP_API int snn_hip_rotary_frequencies(int turned, double base, int scaling,
                                           double factor, double context,
                                           double low, double high,
                                           double* frequencies);

/* Linear attention with a decay for each head: a state of keys x values floats
 * for each head of each sequence,
 *
 *   S_t = a S_{t-1} + k_t^T v_t        a = exp(decay[head])
 *   o_t = scale q_t S_t
 *
 * q and k are [batch][steps][key_heads][keys], v and output
 * [batch][steps][heads][values]; heads is a multiple of key_heads, and head h reads
 * the queries and keys of head h / (heads / key_heads).  q, k and v have row
 * strides of their own, elements from step to step (steps times that from sequence
 * to sequence), so that they may be slices of one projection's rows; output has
 * none.  decay holds `heads` floats, logarithms: 0 for a state that keeps
 * everything; values above 0 are taken as 0, values below -10000 as -10000.  Powers
 * of a decay are held above zero, by 2^-126, so that what is infinite stays so.
 * Decays are constants of the model and have no gradient here.
 *
 * initial_state and final_state are [batch][heads][keys][values] floats (NULL: zero,
 * not wanted) and may be one buffer: a single token is a call with one step that
 * updates the state in place.  resets ([batch][steps] bytes, NULL: none): where it
 * is not zero a S_{t-1} is left out, whatever it is.  lengths ([batch] ints, NULL:
 * all steps; clamped to 0 ... steps): steps from there on are not read, their
 * outputs are zero, and final_state is the state behind the last step that counts
 * (the initial state for a length of zero).  Outputs of a step depend on no later
 * step and on no step in front of a reset, whatever values those hold.
 *
 * A few steps are taken one after the other, more in blocks: of each block of steps
 * the products q_t k_s, weighted by their decays, and the states come from the
 * matrix instructions.  These take scale q_t k_s rounded to the data type (in
 * binary16: infinite beyond 65504, in steps of 2^-24 below 2^-14), states as sums of two
 * values of the data type and weighted values as sums of two of binary16, at a range for
 * each of the values' channels in a block, or three of bfloat16; sums and states are
 * fp32.  Long sequences are divided into pieces that run beside one another, given
 * a workspace of the recommended size.  The order of operations is fixed by the sizes and the
 * workspace.  At most 256 channels of a key or a value; more than 2^30 steps, 2^20
 * heads of all sequences or 2^22 elements from step to step are
 * SNN_HIP_INDEX_EXCEEDED. */
typedef struct snn_hip_linear_attention_params {
  int batch;
  int steps;
  int heads;     /* of values, states, decays and outputs */
  int key_heads; /* of queries and keys */
  int keys;      /* channels of a query or key */
  int values;    /* channels of a value */
  int q_stride;
  int k_stride;
  int v_stride;
  int grad_q_stride;
  int grad_k_stride;
  int grad_v_stride;
  float scale;
} snn_hip_linear_attention_params;
SNN_HIP_API int snn_hip_linear_attention_f32(
    const void* q, const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* output, float* final_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_attention_f16(
    const void* q, const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* output, float* final_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_attention_bf16(
    const void* q, const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* output, float* final_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* The gradients.  grad_final_state may be NULL.  grad_q, grad_k and grad_v have
 * strides of their own and are zero from a sequence's length on; each of the four
 * outputs may be NULL and is then not computed.  No output may overlap an input.
 * Where key_heads is not heads, the sums over the heads that share a query or key
 * take workspace: SNN_HIP_INSUFFICIENT_WORKSPACE without the required size; more than
 * 2^23 channels of all heads' keys are then SNN_HIP_INDEX_EXCEEDED. */
SNN_HIP_API int snn_hip_linear_attention_grad_f32(
    const void* grad_output, const float* grad_final_state, const void* q,
    const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* grad_q, void* grad_k, void* grad_v, float* grad_initial_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_attention_grad_f16(
    const void* grad_output, const float* grad_final_state, const void* q,
    const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* grad_q, void* grad_k, void* grad_v, float* grad_initial_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
SNN_HIP_API int snn_hip_linear_attention_grad_bf16(
    const void* grad_output, const float* grad_final_state, const void* q,
    const void* k, const void* v, const float* decay,
    const unsigned char* resets, const int* lengths, const float* initial_state,
    void* grad_q, void* grad_k, void* grad_v, float* grad_initial_state,
    const snn_hip_linear_attention_params* params, void* workspace,
    size_t workspace_elems, void* stream);
/* Workspace of the forward call (grad == 0) or of the gradients, in elements of
 * `dtype`; the forward call requires none. */
SNN_HIP_API int snn_hip_linear_attention_workspace_size(
    const snn_hip_linear_attention_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems);
/* Diagnostics for tests of the kernels: how a call, or one for all four gradients, goes
 * over its sequences in blocks, given a workspace of `workspace_elems` and operands that
 * start at multiples of 16 bytes or do not.  No launches: step by step. */
typedef struct snn_hip_linear_attention_launch {
  int outputs;     /* 1: outputs, 0: the states of pieces */
  int keys;        /* channels of the states' first side, rounded up to 64, 128, 256 */
  int waves;       /* of a work-group */
  int ring;        /* blocks in a ring that rows go to straight; 0: by registers */
  int work_groups;
} snn_hip_linear_attention_launch;
typedef struct snn_hip_linear_attention_plan {
  int pieces;      /* of a sequence */
  int piece_steps;
  int launches;
  snn_hip_linear_attention_launch launch[4];
} snn_hip_linear_attention_plan;
SNN_HIP_API int snn_hip_linear_attention_planned(
    const snn_hip_linear_attention_params* params, int grad, int dtype,
    int aligned, size_t workspace_elems, snn_hip_linear_attention_plan* plan);

#ifdef __cplusplus
}
#endif
#endif /* SNN_HIP_H_ */

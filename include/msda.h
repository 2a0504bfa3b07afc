/*
 * msda.h — C ABI of the MI355X (gfx950) multi-scale deformable-attention library.
 *
 * The library computes RF-DETR-JAX's deformable-attention core: bilinear, zero-padded sampling of
 * a multi-level value map at per-query sample positions, weighted by per-sample attention weights
 * and summed over levels x points; and the three gradients of that map (value, sampling
 * locations, attention weights).
 *
 * Reference interface replaced (paths are into the RF-DETR-JAX source tree):
 *   msda_fwd  <- ms_deform_attn_core_rows(value, spatial_shapes, sampling_locations,
 *                attention_weights, sampler)            src/rfdetr_jax/models/ops.py:208-292
 *                (the per-level sampler _sample_rows,   ops.py:64-134, and the point-weighted
 *                einsum,                                ops.py:289)
 *   msda_bwd  <- the VJP of the same function, which the reference obtains by JAX autodiff of
 *                ops.py:64-134 + ops.py:289, and which its fused TPU sampler implements by hand
 *                in _sample_bwd / _backward_kernel      src/rfdetr_jax/models/deform_pallas.py:97-120,157-175
 *
 * Layouts (all row-major, contiguous):
 *   value                 [batch * n_heads, len_value, head_dim]    value_dtype   (ops.py:218)
 *   sampling_locations    [batch, len_query, n_heads, n_levels, n_points, 2]  f32, (x, y) in [0,1]
 *   attention_weights     [batch, len_query, n_heads, n_levels * n_points]    f32, level-major
 *   output                [batch, len_query, n_heads * head_dim]    output_dtype  (ops.py:229)
 *   spatial_shapes        host int32 [n_levels][2] = (H_l, W_l)
 *   level_start_index     host int32 [n_levels] = prefix sums of H_l * W_l (may be NULL)
 *   len_value             sum over levels of H_l * W_l
 *
 * Semantics: torch grid_sample(mode="bilinear", padding_mode="zeros", align_corners=False) on the
 * normalised grid 2*loc-1, exactly as ops.py:83-134 and ops.py:270 state it. Sample coordinates
 * are computed in f32 without fused multiply-adds so floor() decisions match the reference.
 *
 * Calls are enqueue-only on `stream` (a hipStream_t, passed as void*; NULL = default stream):
 * no allocation, no host synchronisation, no global mutable state beyond one-time per-device
 * initialisation. All buffers, including the backward's scratch workspace, are owned by the
 * caller. Inputs are read-only; every output element is written by the call (grad_value needs no
 * zero-initialisation).
 *
 * Return values: MSDA_OK (0) or a negative MSDA_ERR_* code; msda_last_error() then returns a
 * message for the calling thread. Argument validation happens before any HIP call.
 */
#ifndef MSDA_H_
#define MSDA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum msda_dtype {
  MSDA_DTYPE_F32 = 0,
  MSDA_DTYPE_BF16 = 1
};

enum msda_status {
  MSDA_OK = 0,
  MSDA_ERR_INVALID_ARGUMENT = -1, /* shapes, pointers or level table inconsistent */
  MSDA_ERR_UNSUPPORTED = -2,      /* valid but outside what the kernels handle (dtype, head_dim) */
  MSDA_ERR_LAUNCH = -3,           /* a kernel launch failed */
  MSDA_ERR_DEVICE = -4            /* a HIP runtime query failed */
};

/*
 * The reference's sampler names (ms_deform_attn_core_rows's `sampler`, ops.py:208-241), for
 * msda_fwd_sampler / msda_bwd_sampler. MSDA_SAMPLER_HIP is this library's own: f32 interpolation
 * throughout, what msda_fwd / msda_bwd compute.
 */
enum msda_sampler {
  MSDA_SAMPLER_HIP = 0,
  MSDA_SAMPLER_GATHER = 1,     /* ops.py:64-134 _sample_rows */
  MSDA_SAMPLER_GATHER_F32 = 2, /* ops.py:137-144 _sample_rows_f32 */
  MSDA_SAMPLER_MATMUL = 3,     /* ops.py:147-186 _sample_rows_matmul */
  MSDA_SAMPLER_AUTO = 4,       /* per level: matmul when H * W <= 4096, else gather (ops.py:42, :277-279) */
  MSDA_SAMPLER_PALLAS = 5      /* deform_pallas.py:193-228 sample_weighted */
};

/* Maximum number of feature levels per call. */
#define MSDA_MAX_LEVELS 16

/* Library version string, e.g. "msda-gfx950 0.1.0". */
const char* msda_version(void);

/* Message describing the last failed call on the calling thread ("" if none). */
const char* msda_last_error(void);

/*
 * Process-wide override of a launch-tuning knob (an MSDA_* name, e.g. "MSDA_BWD_BANDS"); value
 * NULL removes the override. Knobs otherwise come from the environment, read once per name at its
 * first use. They choose launch shapes: results stay within the documented tolerances. The knobs
 * that select the opt-in sorted-gather backward (MSDA_BWD_GATHER*) or force banded backward plans
 * (MSDA_BWD_FORCE_BANDS) change msda_bwd_workspace_size's answer: query it after setting them.
 * Not to be called while another thread launches.
 * No counterpart in the reference; for benchmarks and tests that compare launch variants.
 * Returns MSDA_OK, or MSDA_ERR_INVALID_ARGUMENT for a name that does not start with "MSDA_".
 */
int msda_set_tuning(const char* name, const char* value);

/*
 * Forward: output = sum_{l,p} A[b,q,h,l*P+p] * bilinear(value[b*H+h], level l, loc[b,q,h,l,p]).
 * Replaces ms_deform_attn_core_rows (src/rfdetr_jax/models/ops.py:208-292) and its "pallas"
 * branch (ops.py:243-263 -> deform_pallas.py:193-228 sample_weighted), interpolating in f32
 * throughout; msda_fwd_sampler adds a named sampler's rounding points.
 * output_dtype is the dtype of result_type(value, attention_weights) in the reference (ops.py:260),
 * i.e. MSDA_DTYPE_F32 whenever the weights are f32; MSDA_DTYPE_BF16 is accepted for callers that
 * keep bf16 weights.
 */
int msda_fwd(const void* value, int value_dtype,
             const float* sampling_locations, const float* attention_weights,
             void* output, int output_dtype,
             int batch, int n_heads, int head_dim, int len_query,
             int n_levels, int n_points,
             const int32_t* spatial_shapes, const int32_t* level_start_index,
             int64_t len_value, void* stream);

/*
 * msda_fwd computing what the named reference sampler computes (`sampler`: enum msda_sampler),
 * the `sampler` argument of ms_deform_attn_core_rows (ops.py:208-292). They differ in where a bf16
 * value map is rounded and in how the Pallas kernel forms pixel coordinates; with an f32 value
 * map gather, gather-f32, matmul and auto are the f32 interpolation of msda_fwd.
 *   GATHER      bf16 value: the fractions, 1 - fraction, the four corner-weight products, each
 *               value * weight product and the four-corner sum rounded to bf16 (ops.py:88-91,
 *               :123, :134; the sum taken in f32).
 *   GATHER_F32  bf16 value: f32 interpolation, the sample rounded to bf16 (ops.py:137-144).
 *   MATMUL      bf16 value: the axis kernels 1 - f and f rounded to bf16, their products rounded
 *               to bf16 (ops.py:170-184), the contraction with the values in f32 and rounded to
 *               bf16 (ops.py:186).
 *   AUTO        per level, MATMUL when H * W <= 4096, else GATHER (ops.py:42, :277-279).
 *   PALLAS      pixel coordinates loc * size - 0.5 (deform_pallas.py:223-224) instead of
 *               ((2 loc - 1 + 1) size - 1) / 2 (ops.py:83-84, :270); f32 interpolation.
 * Each sample's weighted sum over levels and points is formed in f32 (ops.py:289). Returns
 * MSDA_ERR_INVALID_ARGUMENT for an unknown sampler code; otherwise as msda_fwd.
 */
int msda_fwd_sampler(const void* value, int value_dtype,
                     const float* sampling_locations, const float* attention_weights,
                     void* output, int output_dtype, int sampler,
                     int batch, int n_heads, int head_dim, int len_query,
                     int n_levels, int n_points,
                     const int32_t* spatial_shapes, const int32_t* level_start_index,
                     int64_t len_value, void* stream);

/*
 * Device workspace msda_bwd needs for this shape, in bytes, or a negative MSDA_ERR_* code: the f32
 * partial grad_value sums of the query blocks when the backward splits each (slice, level)'s
 * queries over several workgroups (n_blocks * batch * n_heads * len_value * head_dim * 4 bytes),
 * else 0. It depends on the shape, the device and the MSDA_* tuning knobs in force (read from the
 * environment once, or set by msda_set_tuning); with no knob set, on the shape and the device
 * only. The reference has no counterpart: JAX autodiff materialises its own intermediates
 * (ops.py:120-134); an XLA FFI handler asks ffi::ScratchAllocator for this many bytes.
 */
int64_t msda_bwd_workspace_size(int batch, int n_heads, int head_dim, int len_query,
                                int n_levels, int n_points,
                                const int32_t* spatial_shapes, const int32_t* level_start_index,
                                int64_t len_value);

/*
 * Backward (vector-Jacobian product of msda_fwd with cotangent grad_output):
 *   grad_value              [batch*n_heads, len_value, head_dim]  value_dtype (accumulated in f32,
 *                           rounded once; deform_pallas.py:175 casts the same way)
 *   grad_sampling_locations [batch, len_query, n_heads, n_levels, n_points, 2] f32
 *   grad_attention_weights  [batch, len_query, n_heads, n_levels*n_points]     f32
 * Replaces the JAX autodiff VJP of ops.py:64-134/289 and deform_pallas.py:157-175 (_sample_bwd).
 * Any of the three gradient pointers may be NULL to skip that gradient. grad_output has
 * grad_output_dtype (the forward's output dtype). grad_value is accumulated in LDS in f64 (a * w of
 * two f32 values is exact in f64, its product with g is rounded to f64's 53 bits); a workgroup owns
 * a (slice, level band) and writes its
 * rows once, rounded to value_dtype, or, when a level's queries are split over several
 * workgroups, writes f32 partial rows into the workspace that a second kernel adds in block order.
 * workspace must hold msda_bwd_workspace_size() bytes (16-byte aligned); it may be NULL when that
 * size is 0 or grad_value is NULL.
 * Limits (MSDA_ERR_UNSUPPORTED beyond them): levels of at most 32000 rows and columns,
 * len_query * n_heads * head_dim < 2^30 and len_query * n_heads * n_levels * n_points < 2^24, and
 * one image row of every level (its f64 accumulator, two staged value rows and a point list of at
 * least one query) within the LDS: about 158 columns at head_dim 64 and 318 at head_dim 32 in f32.
 */
int msda_bwd(const void* value, int value_dtype,
             const float* sampling_locations, const float* attention_weights,
             const void* grad_output, int grad_output_dtype,
             void* grad_value, float* grad_sampling_locations, float* grad_attention_weights,
             int batch, int n_heads, int head_dim, int len_query,
             int n_levels, int n_points,
             const int32_t* spatial_shapes, const int32_t* level_start_index,
             int64_t len_value, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * msda_bwd for the gradient of msda_fwd_sampler: the VJP of the f32 interpolation at the pixel
 * coordinates the named sampler forms (PALLAS: loc * size - 0.5, deform_pallas.py:157-175; the
 * others those of ops.py:83-84), so the floor decisions are the forward's. The bf16 rounding points
 * of GATHER, GATHER_F32 and MATMUL are forward-only: their VJP through the bf16 casts rounds the
 * cotangents and scatter-adds them in bf16 in an order XLA chooses, which no fixed-order kernel
 * reproduces; the gradients here are the f32 ones, within the bf16 tolerance of the reference's.
 * Workspace as msda_bwd_workspace_size(); arguments and results otherwise as msda_bwd.
 */
int msda_bwd_sampler(const void* value, int value_dtype,
                     const float* sampling_locations, const float* attention_weights,
                     const void* grad_output, int grad_output_dtype,
                     void* grad_value, float* grad_sampling_locations, float* grad_attention_weights,
                     int sampler,
                     int batch, int n_heads, int head_dim, int len_query,
                     int n_levels, int n_points,
                     const int32_t* spatial_shapes, const int32_t* level_start_index,
                     int64_t len_value, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * msda_bwd without a workspace argument and without any device allocation, for callers that
 * cannot allocate (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). No counterpart in the reference. The partial sums go to a file-scope device array of
 * 16 MiB that the library holds on every GPU it runs on until the process ends; a shape whose
 * msda_bwd_workspace_size() exceeds it returns MSDA_ERR_UNSUPPORTED. Every call on one GPU uses
 * that GPU's array: calls that overlap on one GPU (different streams, or threads) race. Nothing in
 * the array needs clearing (every partial element is written before it is read). Arguments and
 * results otherwise as msda_bwd.
 */
int msda_bwd_noalloc(const void* value, int value_dtype,
                     const float* sampling_locations, const float* attention_weights,
                     const void* grad_output, int grad_output_dtype,
                     void* grad_value, float* grad_sampling_locations, float* grad_attention_weights,
                     int batch, int n_heads, int head_dim, int len_query,
                     int n_levels, int n_points,
                     const int32_t* spatial_shapes, const int32_t* level_start_index,
                     int64_t len_value, void* stream);

/*
 * The MSDeformAttn prologue fused into the kernels. These entry points take what the module's
 * projections produce and form the core's inputs inside the kernels, so sampling locations and
 * attention weights never exist in memory:
 *   sampling_locations = reference_points + sampling_offsets / (W_l, H_l)        (ref_dim == 2)
 *                      = ref[..., :2] + sampling_offsets / n_points * ref[..., 2:] * 0.5
 *                                                                                 (ref_dim == 4)
 *   attention_weights  = softmax(attention_logits) over the n_levels * n_points axis, in f32.
 * Replaces the body of MSDeformAttn.__call__ from the offsets to the core call,
 * src/rfdetr_jax/models/ops.py:388-410 (locations :388-399 with precise_divide :46-62, softmax
 * :403-404, core :408-410), and its JAX autodiff VJP.
 * Layouts:
 *   reference_points  [batch, len_query, n_levels, ref_dim]                     f32 (ref_dim 2 or 4)
 *   sampling_offsets  [batch, len_query, n_heads, n_levels, n_points, 2]         f32
 *   attention_logits  [batch, len_query, n_heads, n_levels * n_points]           f32
 * Other arguments as msda_fwd; reference_points must be aligned to 4 * ref_dim bytes.
 */
int msda_fused_fwd(const void* value, int value_dtype,
                   const float* reference_points, int ref_dim,
                   const float* sampling_offsets, const float* attention_logits,
                   void* output, int output_dtype,
                   int batch, int n_heads, int head_dim, int len_query,
                   int n_levels, int n_points,
                   const int32_t* spatial_shapes, const int32_t* level_start_index,
                   int64_t len_value, void* stream);

/*
 * Workspace of msda_fused_bwd, in bytes, or a negative MSDA_ERR_* code: msda_bwd's record bins
 * plus per-head-group partial sums of the reference-point gradient (up to
 * batch * len_query * n_heads * n_levels * ref_dim floats), summed by a small second kernel.
 */
int64_t msda_fused_bwd_workspace_size(int batch, int n_heads, int head_dim, int len_query,
                                      int n_levels, int n_points, int ref_dim,
                                      const int32_t* spatial_shapes, const int32_t* level_start_index,
                                      int64_t len_value);

/*
 * Backward of msda_fused_fwd:
 *   grad_value              [batch*n_heads, len_value, head_dim]   value_dtype
 *   grad_sampling_offsets   [batch, len_query, n_heads, n_levels, n_points, 2]  f32
 *   grad_attention_logits   [batch, len_query, n_heads, n_levels*n_points]      f32
 *   grad_reference_points   [batch, len_query, n_levels, ref_dim]               f32
 * Any gradient pointer may be NULL to skip it. The workspace (16-byte aligned, at least
 * msda_fused_bwd_workspace_size() bytes) is needed when grad_value or grad_reference_points is
 * requested. Limits as msda_bwd.
 */
int msda_fused_bwd(const void* value, int value_dtype,
                   const float* reference_points, int ref_dim,
                   const float* sampling_offsets, const float* attention_logits,
                   const void* grad_output, int grad_output_dtype,
                   void* grad_value, float* grad_sampling_offsets, float* grad_attention_logits,
                   float* grad_reference_points,
                   int batch, int n_heads, int head_dim, int len_query,
                   int n_levels, int n_points,
                   const int32_t* spatial_shapes, const int32_t* level_start_index,
                   int64_t len_value, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Grid sampling of channels-first feature maps: bilinear_grid_sample and point_sample of the
 * segmentation head. Replaces
 *   bilinear_grid_sample(inputs, grid, padding_mode)   src/rfdetr_jax/models/ops.py:189-205
 *     (the sampler _sample_rows with padding_mode,    ops.py:64-134)
 *   point_sample(inputs, point_coords, mode)           src/rfdetr_jax/models/heads/segmentation.py:146-170
 *     (nearest sampling, _nearest_grid_sample,         segmentation.py:173-186)
 * and their JAX autodiff VJPs.
 * Layouts (row-major, contiguous):
 *   input        [n, channels, height, width]   dtype (MSDA_DTYPE_F32 or MSDA_DTYPE_BF16)
 *   grid         [n, n_points, 2] f32 (x, y): grid coordinates in [-1, 1] (MSDA_GRID_COORDS,
 *                bilinear_grid_sample; n_points = Hg * Wg) or point_sample's points in [0, 1]
 *                (MSDA_GRID_UNIT_POINTS; the kernel forms grid = 2 p - 1, segmentation.py:166)
 *   output       [n, channels, n_points]        dtype
 * Semantics: torch grid_sample(align_corners=False) as ops.py:64-134 writes it; zero padding masks
 * out-of-bounds corners, border padding clips them (the unmasked weights replicate the edge);
 * nearest sampling rounds half to even and clips, with border padding only.
 */
enum msda_grid_kind { MSDA_GRID_COORDS = 0, MSDA_GRID_UNIT_POINTS = 1 };
enum msda_padding { MSDA_PADDING_ZEROS = 0, MSDA_PADDING_BORDER = 1 };
enum msda_sample_mode { MSDA_SAMPLE_BILINEAR = 0, MSDA_SAMPLE_NEAREST = 1 };

int msda_grid_sample_fwd(const void* input, int dtype, const float* grid, int grid_kind,
                         void* output, int n, int channels, int height, int width, int n_points,
                         int padding_mode, int sample_mode, void* stream);

/*
 * Backward of msda_grid_sample_fwd for cotangent grad_output [n, channels, n_points] (dtype):
 *   grad_input [n, channels, height, width] dtype (accumulated in f32, fully written: no
 *              zero-fill needed), and grad_grid [n, n_points, 2] f32 (the gradient of the grid
 *              coordinates or of the unit points, per grid_kind; zero for nearest sampling).
 * Either output may be NULL. Widths above 16384 are MSDA_ERR_UNSUPPORTED for grad_input.
 */
int msda_grid_sample_bwd(const void* input, int dtype, const float* grid, int grid_kind,
                         const void* grad_output, void* grad_input, float* grad_grid,
                         int n, int channels, int height, int width, int n_points,
                         int padding_mode, int sample_mode, void* stream);

/*
 * MSDeformAttn's value projection with its epilogue fused in: one MFMA product writes
 *   value[(b * n_heads + h) * len_in + s][d] = padded[b, s] ? 0 : (input[b, s, :] . W[h * head_dim + d, :] + bias[h * head_dim + d])
 * Replaces value_proj (Linear, src/rfdetr_jax/models/layers.py:258-280: x @ W^T + b in the input
 * dtype), the padding mask (ops.py:377-379) and the head split (ops.py:405-407) of
 * MSDeformAttn.__call__, so the [B, S, C] projection and its transpose never exist in memory.
 * Layouts:
 *   input         [batch, len_in, in_features]           dtype (MSDA_DTYPE_F32 or MSDA_DTYPE_BF16)
 *   weight        [n_heads * head_dim, in_features] f32  (torch Linear layout; rounded to bf16 when
 *                                                        the input is bf16, as weight.astype(x.dtype))
 *   bias          [n_heads * head_dim] f32 or NULL
 *   padding_mask  [batch, len_in] uint8 (non-zero = padded) or NULL
 *   value         [batch * n_heads, len_in, head_dim]    dtype (the core's value layout)
 */
int msda_value_proj_fwd(const void* input, int dtype, const float* weight, const float* bias,
                        const uint8_t* padding_mask, void* value,
                        int batch, int len_in, int in_features, int n_heads, int head_dim, void* stream);

/* Workspace of msda_value_proj_bwd in bytes (a function of the shape only), or a negative code. */
int64_t msda_value_proj_bwd_workspace_size(int batch, int len_in, int in_features, int n_heads, int head_dim);

/*
 * Backward of msda_value_proj_fwd for cotangent grad_value [batch * n_heads, len_in, head_dim]:
 *   grad_input  [batch, len_in, in_features] dtype, grad_weight [n_heads * head_dim, in_features]
 *   f32, grad_bias [n_heads * head_dim] f32; padded rows contribute nothing. Any of the three may be
 * NULL. The workspace (16-byte aligned) holds grad_weight's split partial sums and is needed when
 * grad_weight or grad_bias is requested; they are added in a fixed order (deterministic).
 */
int msda_value_proj_bwd(const void* input, int dtype, const float* weight, const uint8_t* padding_mask,
                        const void* grad_value, void* grad_input, float* grad_weight, float* grad_bias,
                        int batch, int len_in, int in_features, int n_heads, int head_dim,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* ---- Decoder self-attention -----------------------------------------------------------------
 * scaled_dot_product_attention (src/rfdetr_jax/models/layers.py:54-99, the XLA path) as used by
 * MultiheadAttention (layers.py:491-548) in the decoder's grouped self-attention
 * (src/rfdetr_jax/models/transformer.py:200-210): per slice z and head h,
 *   out = softmax(q k^T / sqrt(D), blocked positions -> finfo(float32).min) v
 * over len queries and len keys of head_dim = D channels (32 or 64). The slices are
 * z = g * batch + b for b < batch, g < groups, the order of _split_groups (transformer.py:350-354):
 * with groups > 1 the caller passes the unsplit [batch, groups * len, C] rows and the kernels read
 * group g of image b in place. Every tensor is addressed as
 *   base + b * s_b + g * s_g + h * s_h + row * s_row + channel
 * with the four element strides given per tensor in `strides` (in that order; each a multiple of 4,
 * base pointers aligned to 4 elements). Examples: [Z, H, L, D] contiguous (the reference
 * function's layout): (H L D, 0, L D, D) with groups = 1; the decoder's [B, G P, C] rows with
 * C = H D: (G P C, P C, D, C).
 *
 * mask: [len, len] bytes (non-zero blocks a key for a query: torch's boolean convention,
 * layers.py:69, :93-94) or NULL. dtype: MSDA_DTYPE_F32 or MSDA_DTYPE_BF16 for every tensor;
 * sums and softmax are f32. f32 products run on f32 matrix instructions (v_mfma_f32_32x32x2_f32) with
 * a mask or dropout, and otherwise on operands of three bf16 terms, which hold f32's 24 significand
 * bits (attention_split_kernels.h); bf16 products run on bf16 matrix instructions.
 * stats: [batch * groups * heads * len][4] f32, 16-byte aligned, z-major (z = g * batch + b), then
 * head, then query: the forward writes entries 0 and 1, whose sum is log2 of the row's sum of 2^x over
 * the keys, x = log2(e) q.k / sqrt(D) (entry 0 alone is within 64 of that sum); the backward reads them
 * and uses entry 2 for rowsum(grad_out * out).
 * Dropout on the attention weights (layers.py:537-544, active only with dropout > 0 in training)
 * is msda_attention_fwd_dropout's. len is at most 65536, each row stride s_row below 2^24 elements
 * and len * s_row below 2^31 (row offsets within a (slice, head) are formed in 32 bits).
 */
int msda_attention_fwd(const void* q, const void* k, const void* v, int dtype, void* out, float* stats,
                       int batch, int groups, int heads, int len, int head_dim,
                       const int64_t* strides /* [4 tensors: q, k, v, out][4] */, const uint8_t* mask, void* stream);

/*
 * Backward of msda_attention_fwd for the cotangent grad_out: grad_q, grad_k, grad_v (each may be
 * NULL to skip it; same layouts and dtype rules). out and stats are the forward's (stats entry 2
 * is overwritten). With head_dim 32, no mask, len <= 320 and grad_q plus grad_k or grad_v
 * requested, one kernel forms all gradients (the tuning knob MSDA_ATTN_FUSED=0 selects the
 * two-kernel path instead; the two agree within f32 summation order).
 * strides: [8 tensors: q, k, v, out, grad_out, grad_q, grad_k, grad_v][4].
 */
int msda_attention_bwd(const void* q, const void* k, const void* v, const void* out, float* stats,
                       const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v,
                       int batch, int groups, int heads, int len, int head_dim,
                       const int64_t* strides, const uint8_t* mask, void* stream);

/*
 * msda_attention_fwd with dropout on the softmax weights, as MultiheadAttention applies it in
 * training (layers.py:537-544: weights = nn.Dropout(rate)(softmax(scores)), then weights @ v):
 *   out = (softmax(...) * keep / (1 - rate)) v.
 * keep(z, h, q, k) is a function of (seed, z * heads + h, q, k) alone: each kernel that needs it
 * regenerates it, so the backward of the same call (same seed and rate) drops the same weights and
 * nothing is stored. A weight is kept with probability 1 - round(rate * 65536) / 65536. The
 * reference draws its mask from JAX's threefry stream (flax nn.Dropout): the distribution is the
 * same, the particular mask is not. rate in [0, 1) (MSDA_ERR_INVALID_ARGUMENT otherwise); rate 0
 * computes what msda_attention_fwd computes. stats as msda_attention_fwd's (the softmax of every
 * weight, before dropout). Dropout runs in the chunked kernels (neither the staged bf16 forward nor
 * the fused backward).
 * No counterpart in the reference's C interface (its dropout is a JAX op around the product); for
 * callers that train with attention dropout.
 */
int msda_attention_fwd_dropout(const void* q, const void* k, const void* v, int dtype, void* out, float* stats,
                               int batch, int groups, int heads, int len, int head_dim,
                               const int64_t* strides, const uint8_t* mask, float rate, uint64_t seed, void* stream);

/*
 * Backward of msda_attention_fwd_dropout (same rate and seed as the forward call):
 *   dV = (P * keep / (1 - rate))^T dO,  dP = (dO V^T) * keep / (1 - rate),
 *   dS = P (dP - rowsum(dO * out)),     dQ = dS K / sqrt(D),  dK = dS^T Q / sqrt(D).
 * Arguments otherwise as msda_attention_bwd (always the two-kernel path).
 */
int msda_attention_bwd_dropout(const void* q, const void* k, const void* v, const void* out, float* stats,
                               const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v,
                               int batch, int groups, int heads, int len, int head_dim,
                               const int64_t* strides, const uint8_t* mask, float rate, uint64_t seed, void* stream);

/*
 * The keep decisions of msda_attention_fwd_dropout for (rate, seed): keep[z * heads + h][q][k] = 1
 * where weight (q, k) is kept, else 0 ([batch * groups * heads][len][len] bytes, z = g * batch + b).
 * For tests and for callers that need the mask itself; no counterpart in the reference.
 */
int msda_attention_dropout_keep(int batch, int groups, int heads, int len, float rate, uint64_t seed,
                                uint8_t* keep, void* stream);

/* ---- Attention over packed sequences --------------------------------------------------------
 * Softmax attention of sequences of different lengths that lie behind one another, with fewer key
 * heads than query heads (heads a multiple of kv_heads: query head h reads key head
 * h / (heads / kv_heads)), causal or not. No counterpart in the reference, whose attention
 * (layers.py:54-99) takes one length, one number of heads and an explicit mask.
 *   q, out, grad_out, grad_q   [q_rows, heads, head_dim]       dtype
 *   k, v, grad_k, grad_v       [k_rows, kv_heads, head_dim]    dtype
 *   q_offsets, k_offsets       [sequences + 1] int32, device memory, rising
 *   k_lengths                  [sequences] int32, device memory, or NULL
 * Sequence i holds the query rows q_offsets[i] .. q_offsets[i + 1] - 1 (n of them) and the m key rows
 * from k_offsets[i] on: as many as k_lengths[i] says, or all before k_offsets[i + 1] (a cache has room
 * for more rows than it holds). Query t of a sequence sees its keys j < m, with `causal` those with
 * j <= t + m - n: the last query sees every key, so one new token over a cache of m keys is n = 1.
 *   out = softmax(scale q k^T over the seen keys) v, 0 where no key is seen.
 * A pair that is not seen takes no part, whatever its rows hold (infinities and NaN too). Rows of out and of the gradients that
 * belong to no sequence, and of grad_k and grad_v from the m-th of a sequence on, are written as zeros.
 * Offsets and lengths are clamped to the tensors' rows: others than rising ones give unspecified
 * values, never an access out of bounds.
 *
 * head_dim: a multiple of 8, at most 128. `strides` holds the element strides (row, head) of each
 * tensor (0, 0 for one that is NULL); channels are contiguous, and rows start on 16-byte boundaries (bases, and strides in bytes, are
 * multiples of 16), head_dim to 2^22 elements apart, q's and grad_out's heads of a key head within
 * 2^27 elements. At most 64 query heads to a key head; backward: fewer than 2^21 key heads. scale: 2^-64 to 2^64.
 * q_rows * heads / kv_heads and k_rows below 2^31 less 128 rows a sequence.
 * stats: [q_rows * heads][4] f32, 16-byte aligned: the forward writes entries 0 and 1 (their sum is log2
 * of the row's sum of 2^(scale2 q.k), scale2 = scale log2(e)), the backward reads them. May be NULL in a forward whose backward is not wanted.
 * out_rest: NULL, or for bf16 a tensor of out's strides: the forward writes what out's rounding left, the
 * backward reads out + out_rest for rowsum(grad_out * out), whose error is then that of f32 sums.
 * Sums, softmax and statistics are f32; f32 products run on f32 matrix instructions, bf16 ones on bf16 matrix
 * instructions, with the softmax weights and their gradients rounded to bf16. The weights of out keep two bf16
 * numbers where a sequence's queries times heads / kv_heads are at most 32, and, as grad_q's gradients of
 * weights, where a row sees fewer than 64 keys. No result depends on an order of atomics.
 */

/*
 * Device workspaces in bytes (functions of the shape only), or a negative code; 0 where nothing is split.
 * Forward: partial sums of calls whose keys are split over several workgroups, because few query rows (of
 * which there are at most 32 a sequence on average) stand over long ranges of keys, or because the tiles of
 * 128 rows do not fill the CUs evenly (prompts, too: one f32 sequence of 4,096 tokens, 8 heads, 128 channels,
 * 307 MB for an output of 17). (parts (head_dim + 2) + 1) q_rows heads 4 with parts <= 64.
 * Backward: partial sums of grad_k and grad_v where there are so few key tiles that the rows seeing one are
 * split: parts 2 k_rows kv_heads head_dim 4 with parts <= 8, room for all rows though few tiles may have
 * parts: up to 16 times the two gradients in bf16, 8 times in f32.
 */
int64_t msda_packed_attention_fwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim);
int64_t msda_packed_attention_bwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim);

/* strides: [4 tensors: q, k, v, out][2]. The workspace is 16-byte aligned; NULL when its size is 0. */
int msda_packed_attention_fwd(const void* q, const void* k, const void* v, int dtype, void* out, void* out_rest,
                              float* stats, const int32_t* q_offsets, const int32_t* k_offsets,
                              const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads,
                              int kv_heads, int head_dim, const int64_t* strides, int causal, float scale,
                              void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Backward of msda_packed_attention_fwd for the cotangent grad_out: grad_q, grad_k, grad_v (each may be
 * NULL to skip it). out, out_rest and stats are the forward's. Entries 2 and 3 of stats are overwritten: two calls
 * with one stats have to come one behind the other (msda_packed_attention_bwd_const otherwise).
 * strides: [8 tensors: q, k, v, out, grad_out, grad_q, grad_k, grad_v][2].
 */
int msda_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest,
                              float* stats, const void* grad_out, int dtype, void* grad_q, void* grad_k,
                              void* grad_v, const int32_t* q_offsets, const int32_t* k_offsets,
                              const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads,
                              int kv_heads, int head_dim, const int64_t* strides, int causal, float scale,
                              void* workspace, int64_t workspace_bytes, void* stream);

/*
 * The same with stats left as they are. row_numbers: [q_rows * heads][4] f32, 16-byte aligned, which the call
 * uses between its kernels (NULL when neither grad_k nor grad_v is wanted).
 */
int msda_packed_attention_bwd_const(const void* q, const void* k, const void* v, const void* out, const void* out_rest,
                                    const float* stats, float* row_numbers, const void* grad_out, int dtype,
                                    void* grad_q, void* grad_k, void* grad_v, const int32_t* q_offsets,
                                    const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows,
                                    int k_rows, int heads, int kv_heads, int head_dim, const int64_t* strides,
                                    int causal, float scale, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Attention over packed sequences with shaped scores. Query t of a sequence stands at the place t + m - n among its
 * keys. Its score for key j is
 *   x = cap tanh(scale q.k / cap) - slopes[head] |place - j|
 * (without cap: scale q.k), and it sees the keys with |place - j| < window and, where causal, j <= place or
 * j < prefix_lengths[sequence]; everything else is as above, stats included (log2 of the sum of 2^(x log2(e))).
 * cap: 0 (none) or 2^-32 to 2^32. window: 0 (none) or the number of places. slopes: [heads] f32, device memory, finite,
 * or NULL. prefix_lengths: [sequences] int32, device memory, or NULL; only with causal (a sequence's first keys, which
 * all its queries see: a prompt or an image before a text; 0 and less: none).
 * shape NULL: the calls above. A window makes keys, tiles and the work that lie outside it go away.
 * Backward: msda_packed_attention_bwd_const's arguments. slopes have no gradient.
 * Workspaces: as above, with the window (0: none); the backward's holds partial sums of grad_q, too, where the tiles of
 * queries are fewer than the CUs.
 */
typedef struct msda_score_shape {
  float cap;
  int window;
  const float* slopes;
  const int32_t* prefix_lengths;
} msda_score_shape;

int64_t msda_packed_attention_shaped_fwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                                                        int head_dim, int window);
int64_t msda_packed_attention_shaped_bwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                                                        int head_dim, int window);

int msda_packed_attention_shaped_fwd(const void* q, const void* k, const void* v, int dtype, void* out, void* out_rest,
                                     float* stats, const int32_t* q_offsets, const int32_t* k_offsets,
                                     const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads,
                                     int kv_heads, int head_dim, const int64_t* strides, int causal, float scale,
                                     const msda_score_shape* shape, void* workspace, int64_t workspace_bytes, void* stream);

int msda_packed_attention_shaped_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest,
                                     const float* stats, float* row_numbers, const void* grad_out, int dtype,
                                     void* grad_q, void* grad_k, void* grad_v, const int32_t* q_offsets,
                                     const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows,
                                     int k_rows, int heads, int kv_heads, int head_dim, const int64_t* strides, int causal,
                                     float scale, const msda_score_shape* shape, void* workspace, int64_t workspace_bytes,
                                     void* stream);

/* ---- A cache of keys and values in 4 bits ----------------------------------------------------
 * For serving: rows of keys and values held in 4.25 bits a channel, the calls that write and read rows, and attention
 * over them. No counterpart in the reference.
 *   codes  (keys, values)                [kv_heads, rows, 16 B] bytes, B = ceil(head_dim / 32), 16-byte aligned
 *   scales (key_scales, value_scales)    [kv_heads, rows, B] bytes
 * 32 channels of a row are a block with one power of two 2^e, held as e + 127; a channel is 4 bits, the first of two in
 * the lower half of their byte: a sign (8) and the code of {0, 1/2, 1, 3/2, 2, 3, 4, 6} times 2^e. Writing takes the least
 * e with every magnitude within 7 2^e, from -120 to 125, and the nearest value for each channel, the even code between
 * two. A block that holds an infinity or NaN reads as NaN (scale 255; 253 and 254, which no block gets, too). Channels behind head_dim are zeros.
 *
 * Sequences as above: sequence i's keys are the rows from k_offsets[i] on, as many as k_lengths[i] says (NULL: all before
 * k_offsets[i + 1]), and its tokens q_offsets[i] .. q_offsets[i + 1] - 1 are the newest of them: its last token is its
 * last key. msda_cache4_write puts the tokens' keys and values there (k_lengths counts them already),
 * msda_cache4_read gives the values that the rows there stand for, in dtype (exact in both). Tokens of no sequence, and
 * those older than its keys, are not written, and read as zeros; other rows of the cache stay as they are. Sequences whose
 * rows overlap write over each other in no order. k, v: [tokens, kv_heads, head_dim], strides [2][2] in elements (token,
 * head), channels contiguous, rows on 16-byte boundaries; tokens ceil(kv_heads B / 8) < 2^26.
 *
 * msda_cache4_attention: msda_packed_attention_shaped_fwd over the cache (shape NULL: plain scores), without statistics;
 * strides of q and out [2][2]. Every value of the cache is a bf16 number exactly; with bf16 queries weights and out are
 * rounded as there (two bf16 numbers a weight for sequences of few rows), f32 queries are f32 throughout. The workspace
 * holds partial sums, as there; its size is 0 where nothing is split.
 */
int msda_cache4_write(const void* k, const void* v, int dtype, uint8_t* keys, uint8_t* key_scales, uint8_t* values,
                      uint8_t* value_scales, const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths,
                      int sequences, int tokens, int rows, int kv_heads, int head_dim, const int64_t* strides, void* stream);

int msda_cache4_read(const uint8_t* keys, const uint8_t* key_scales, const uint8_t* values, const uint8_t* value_scales,
                     void* k, void* v, int dtype, const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths,
                     int sequences, int tokens, int rows, int kv_heads, int head_dim, const int64_t* strides, void* stream);

int64_t msda_cache4_attention_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                                             int head_dim, int window);

int msda_cache4_attention(const void* q, int dtype, void* out, const uint8_t* keys, const uint8_t* key_scales,
                          const uint8_t* values, const uint8_t* value_scales, const int32_t* q_offsets,
                          const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads,
                          int kv_heads, int head_dim, const int64_t* strides, int causal, float scale,
                          const msda_score_shape* shape, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- Rotary positions on several axes -------------------------------------------------------
 * Rotates channel pairs of queries and keys by angles that grow with the token's position on each of
 * `axes` axes (time, height, width, ...). No counterpart in the reference.
 *   q, q_out  [tokens, heads, head_dim], k, k_out  [tokens, kv_heads, head_dim]   dtype
 *   positions [tokens, axes]  int32, int64 or f32 (enum msda_position_type), device memory
 *   sections  host int32 [axes]: the number of pairs of each axis, in order; n is their sum, 2 n <= head_dim
 * Pair i, the j-th of axis a, turns by positions[t][a] * base^-e: with shared_frequencies e = i / n (the
 * axes share one falling sequence), else e = j / sections[a] (each axis has its own). Its channels are
 * (i, i + n), or (2 i, 2 i + 1) with `interleaved`:
 *   (u, w) -> (u cos - w sin, u sin + w cos).
 * Channels from 2 n on are copied. inverse: by the negative angles (the gradient for the cotangents of
 * q_out and k_out). Angles are formed in f64 and reduced to one turn before cos and sin, so that far
 * positions keep their precision; the products are f32, rounded once.
 * strides: element strides (token, head) of q, q_out, k, k_out [4][2], channels contiguous;
 * position_strides: (token, axis). An output may be its input. heads or kv_heads may be 0 (its pointers
 * NULL). head_dim even, at most 256; at most 8 axes.
 */
enum msda_position_type { MSDA_POSITION_I32 = 0, MSDA_POSITION_I64 = 1, MSDA_POSITION_F32 = 2 };

int msda_rotary(const void* q, void* q_out, const void* k, void* k_out, int dtype,
                const void* positions, int position_type, int tokens, int heads, int kv_heads, int head_dim,
                const int64_t* strides, const int64_t* position_strides, const int32_t* sections, int axes,
                double base, int shared_frequencies, int interleaved, int inverse, void* stream);

/* ---- Norms of queries and keys with rotary positions ----------------------------------------
 * Each head of each token, a row x of head_dim channels, becomes R [x r w] with r = 1 / sqrt(mean(x^2) + eps), w the
 * head's weight ([head_dim], the same for all heads of q, of k; NULL: ones) and R the rotation of msda_rotary, whose
 * arguments the others are. Queries and keys take one launch. No counterpart in the reference.
 *   weight_type: enum msda_dtype of the weights and of their gradients, f32 or bf16.
 *   strides: element strides (token, head), forward of q, q_out, k, k_out [4][2]; backward of q, grad_q_out, grad_q, k,
 *   grad_k_out, grad_k [6][2]. An output may be its input.
 * eps: 2^-126 to 2^126. Sums are f32, results rounded once. The forward takes fewer than 2^27 tokens.
 * Backward, for the cotangents of q_out and k_out: grad_q, grad_k and the weights' gradients (each may be NULL), the last
 * as sums over all tokens and heads in a fixed order, which take the workspace (NULL without them).
 */
int msda_norm_rotary_fwd(const void* q, void* q_out, const void* k, void* k_out, int dtype, const void* q_weight, const void* k_weight,
                         int weight_type, const void* positions, int position_type, int tokens, int heads, int kv_heads, int head_dim,
                         const int64_t* strides, const int64_t* position_strides, const int32_t* sections, int axes, double base,
                         int shared_frequencies, int interleaved, double eps, void* stream);

int64_t msda_norm_rotary_bwd_workspace_size(int tokens, int head_dim);

int msda_norm_rotary_bwd(const void* q, const void* grad_q_out, void* grad_q, const void* k, const void* grad_k_out, void* grad_k, int dtype,
                         const void* q_weight, const void* k_weight, void* grad_q_weight, void* grad_k_weight, int weight_type,
                         const void* positions, int position_type, int tokens, int heads, int kv_heads, int head_dim,
                         const int64_t* strides, const int64_t* position_strides, const int32_t* sections, int axes, double base,
                         int shared_frequencies, int interleaved, double eps, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSDA_H_ */

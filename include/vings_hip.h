/*
 * vings_hip.h -- C ABI of libvings_hip.so, the MI355X (gfx950) hot-path core
 * for VINGS-Mono: 2D-Gaussian surfel rasteriser forward/backward, row-masked
 * Adam, and the dense bundle-adjustment (DBA) core.
 *
 * The reference reaches this path through two Python extension modules
 * whose native sources are not vendored:
 *   diff_surfel_rasterization  (/root/reference/scripts/gaussian/gaussian_base.py:5-6)
 *   droid_backends             (/root/reference/scripts/frontend/depth_video.py:4)
 * Each entry point below names the reference call it serves.  The Python
 * drop-in modules in vings_mono_amd/dropin bind these symbols with ctypes.
 *
 * Conventions
 *   - every pointer is a DEVICE pointer unless the name ends in _host
 *   - `stream` is a hipStream_t passed as void* (NULL = default stream)
 *   - tensors are dense, row-major, float32 unless stated
 *   - the caller owns all device memory, including workspaces; no entry point
 *     allocates device memory.  The library itself owns two small host-side
 *     things, both created at first use and kept: a 1 KiB ring of pinned
 *     mailboxes per GPU (vings_surfel_project) and the event pool of
 *     vings_profile_enable.  vings_splat_compact_plan_static uses 128 KiB of static device
 *     memory per GPU
 *   - vings_surfel_project and vings_splat_compact_plan synchronise with the
 *     host (each returns a count the caller needs to size buffers); everything
 *     else is asynchronous on the given stream
 *   - return value 0 = success, negative = vings_status
 */
#ifndef VINGS_HIP_H
#define VINGS_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum vings_status {
    VINGS_OK = 0,
    VINGS_ERR_ARG = -1,      /* null pointer / bad size */
    VINGS_ERR_HIP = -2,      /* a HIP runtime call failed; see vings_last_error */
    VINGS_ERR_CAPACITY = -3, /* caller-provided buffer too small */
    VINGS_ERR_NUMERIC = -4   /* e.g. Cholesky breakdown */
} vings_status;

/* Human-readable text of the last failure on the calling thread. */
const char* vings_last_error(void);
/* ABI version; bumped when a signature changes. */
int vings_abi_version(void);

#define VINGS_GEOM_STRIDE 24 /* floats per packed splat record (96 B, 16-byte aligned rows) */
#define VINGS_GRAD_STRIDE 20 /* floats per packed splat gradient record */
#define VINGS_AUX_CHANNELS 9 /* allmap channels */
#define VINGS_TILE 16

/* ------------------------------------------------------------------------
 * Surfel rasteriser forward, stage 1: projection + per-splat tile counts.
 * Serves GaussianRasterizer.forward (gaussian_base.py:193-203), settings
 * tuple built at gaussian_base.py:160-177.
 *
 * in : means3D[N,3] scales[N,2] rotations[N,4](w,x,y,z) opacities[N]
 *      colors[N,3] flow[N,2] or NULL; viewmatrix[16] projmatrix[16] as the
 *      flat storage of the reference's transposed matrices (cameras.py:58-60)
 * out: geom[N,24]  packed record {Tu[3], x, Tv[3], y, Tw[3], normal[3], opacity, rgb[3],
 *                  flow[2]} (T = rows of the pixel homography, (x, y) = pixel centre) +
 *                  box[4] = xmin,xmax,ymin,ymax of the pixels the splat can reach with
 *                  alpha >= 1/255 (conservative; lets a wave skip the splat)
 *                  (rows of culled splats are left untouched)
 *      depth[N] radii[N](int32) rect[N,4](int32 x0,y0,x1,y1 in tiles; packed form under tight binning, see vings_surfel_set_tight_binning)
 *      tiles_touched[N](uint32)
 *      block_prefix[3*ceil(N/256)+4] (uint32): the first ceil(N/256)+1 entries are the
 *                  exclusive prefix of per-256-splat instance counts (last = total); the
 *                  rest is scratch for the depth range
 *      *num_instances_host  total number of (splat,tile) instances D
 *      depth_bits_range_host[2] (may be NULL): smallest and largest float bit pattern of
 *                  the depths of the binned splats; hand both to vings_surfel_bin
 * Synchronises `stream` once to return D and the range.
 */
int vings_surfel_project(int N, int H, int W, float scale_modifier,
                         const float* means3D, const float* scales, const float* rotations,
                         const float* opacities, const float* colors, const float* flow,
                         const float* viewmatrix, const float* projmatrix,
                         float* geom, float* depth, int32_t* radii, int32_t* rect,
                         uint32_t* tiles_touched, uint32_t* block_prefix,
                         int64_t* num_instances_host, uint32_t* depth_bits_range_host,
                         void* stream);

/* Which tiles a splat is binned into (process-wide switch, returns the previous value).
 * 0: every tile of the reference's square of side 2*radius about the splat centre (getRect in
 *    the rasteriser's auxiliary.h, called from forward.cu preprocessCUDA): rect, tiles_touched,
 *    the instance count D, keys and ranges are then exactly the reference's.
 * 1 (default): only the tiles of that square which the splat's alpha >= 1/255 footprint
 *    reaches: its pixel box first, then, for rectangles of up to 64 tiles, the conic test the
 *    blend passes apply per 8x8 block.  The blend passes reject the other tiles with the same
 *    tests before they evaluate a pixel, so colour, allmap, radii and all gradients are
 *    unchanged; the instance list is a subset of the reference's list in the same order
 *    (about 40 % shorter on the benchmark scene), n_contrib counts positions in the shorter
 *    list, and rect holds for such a splat {1<<31 | x0 | y0<<15, width, tile bits lo, hi}
 *    (one bit per tile of the rectangle, row-major) instead of {x0, y0, x1, y1}. */
int vings_surfel_set_tight_binning(int on);
/* The same choice for the projections launched by the CALLING THREAD only (1 / 0; -1: follow
 * the process-wide switch again, the initial state); returns the thread's previous value.
 * Threads that render on one GPU with different binning modes do not disturb each other. */
int vings_surfel_set_tight_binning_thread(int mode);

/* The same call in two halves, for callers that do not want the GPU to idle while the host
 * learns D: launch returns at once; wait blocks until the projection launched last on the
 * current GPU BY THE CALLING THREAD has finished (on an event behind it, not on the whole
 * stream) and returns its D and depth-bit range.  Between the two the caller may enqueue more
 * work on the stream, typically vings_surfel_bin_speculative and the blend sized from the
 * previous view's count.  Every launch takes its own mailbox slot and event from a ring of 16
 * per GPU, so threads (and the streams they drive) that render on one GPU at the same time do
 * not disturb each other; a thread's wait always refers to that thread's latest launch. */
int vings_surfel_project_launch(int N, int H, int W, float scale_modifier,
                                const float* means3D, const float* scales,
                                const float* rotations, const float* opacities,
                                const float* colors, const float* flow,
                                const float* viewmatrix, const float* projmatrix,
                                float* geom, float* depth, int32_t* radii, int32_t* rect,
                                uint32_t* tiles_touched, uint32_t* block_prefix, void* stream);
/* vings_surfel_project_launch on the STORED parameters: the kernel applies the mapper's
 * activations itself (scales = exp(raw_scaling), rotations = raw_rotation / max(|.|, 1e-12),
 * opacities = sigmoid(raw_opacity): gaussian_base.py:44-48,64-72; bit-identical to
 * vings_splat_activate) and leaves the activated arrays in scales / rotations / opacities for
 * the backward pass.  Saves the separate activation launch of the mapper's view step.
 * dgeom_clear (optional, [N, VINGS_GRAD_STRIDE]): the rows of the splats with radii > 0 are
 * zeroed, ready for vings_surfel_blend_backward_accumulate (saves the clearing command of the
 * backward pass; rows of culled splats are not touched and never read). */
int vings_surfel_project_launch_activate(
    int N, int H, int W, float scale_modifier, const float* means3D, const float* raw_scaling,
    const float* raw_rotation, const float* raw_opacity, const float* colors, const float* flow,
    const float* viewmatrix, const float* projmatrix, float* scales, float* rotations,
    float* opacities, float* geom, float* depth, int32_t* radii, int32_t* rect,
    uint32_t* tiles_touched, uint32_t* block_prefix, float* dgeom_clear, void* stream);
int vings_surfel_project_wait(int64_t* num_instances_host, uint32_t* depth_bits_range_host);

/* Bytes of scratch vings_surfel_bin needs for D instances. */
size_t vings_surfel_bin_workspace_bytes(int64_t D);

/* ------------------------------------------------------------------------
 * Stage 2: duplicate with keys (tile<<32 | depth bits), order by (tile, depth, splat) - what
 * a stable sort of the instances emitted in splat order gives -, per-tile ranges.  Same
 * reference call as above.
 * out: keys_sorted[D](uint64) vals_sorted[D](uint32 splat index)
 *      ranges[T,2](uint32 begin,end; 8-byte aligned) with T = ceil(W/16)*ceil(H/16)
 * workspace: vings_surfel_bin_workspace_bytes(D) bytes, 256-byte aligned.
 * depth_bits_min/max: the range vings_surfel_project returned; not used any more (the radix
 * passes run over the tile bits only, the depth order is made per tile in LDS), any values do.
 */
int vings_surfel_bin(int N, int H, int W, int64_t D, uint32_t depth_bits_min,
                     uint32_t depth_bits_max, const float* depth, const int32_t* rect,
                     const uint32_t* tiles_touched, const uint32_t* block_prefix,
                     uint64_t* keys_sorted, uint32_t* vals_sorted, uint32_t* ranges,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Stage 2 launched before the host knows D: buffers (keys_sorted, vals_sorted, workspace)
 * hold D_capacity instances and the kernels read the true D from tail[2],
 * tail = block_prefix + 3*ceil(N/256) + 1 of the projection on the same stream.  Nothing is
 * written beyond the capacity and no range reaches beyond it.  The result equals that of
 * vings_surfel_bin iff D <= D_capacity; the caller checks this after
 * vings_surfel_project_wait and otherwise repeats the stage with vings_surfel_bin.
 * low_bits_guess is not used any more (vings_surfel_bin_low_bits: bits needed for the depth
 * range, kept for callers that size things by it). */
int vings_surfel_bin_low_bits(uint32_t depth_bits_min, uint32_t depth_bits_max);
int vings_surfel_bin_speculative(int N, int H, int W, int64_t D_capacity, int low_bits_guess,
                                 const uint32_t* tail, const float* depth, const int32_t* rect,
                                 const uint32_t* tiles_touched, const uint32_t* block_prefix,
                                 uint64_t* keys_sorted, uint32_t* vals_sorted, uint32_t* ranges,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Stage 3: front-to-back alpha blend, one workgroup per 16x16 tile.
 * out: out_color[3,H,W]  allmap[9,H,W] (0 sum w*depth, 1 alpha, 2:5 sum w*normal,
 *      5 median depth, 6 distortion, 7:9 sum w*flow)  -- consumer:
 *      gaussian_base.py:205-219, gaussian_model.py:427
 *      final_T[3,H,W] (T, M1, M2) and n_contrib[2,H,W](uint32) are saved
 *      state for the backward pass.
 * pixel_mask[H*W] (uint8, 0 = skip pixel) may be NULL (gaussian_base.py:158).
 */
int vings_surfel_blend_forward(int H, int W, const uint32_t* ranges, const uint32_t* vals_sorted,
                               const float* geom, const float* bg, const uint8_t* pixel_mask,
                               float* out_color, float* allmap, float* final_T,
                               uint32_t* n_contrib, void* stream);

/* ------------------------------------------------------------------------
 * Backward of stage 3.  Triggered by total_loss.backward()
 * (gaussian_base.py:382).  dgeom[N,20] receives, per splat,
 * {dT[9], dxy[2], dnormal[3], dopacity, drgb[3], score_importance, score_error};
 * it is zeroed by this call.
 */
int vings_surfel_blend_backward(int N, int H, int W, const uint32_t* ranges,
                                const uint32_t* vals_sorted, const float* geom, const float* bg,
                                const uint8_t* pixel_mask, const float* final_T,
                                const uint32_t* n_contrib, const float* dL_dcolor,
                                const float* dL_dallmap, float* dgeom, void* stream);
/* The same pass ADDING into dgeom instead of clearing it first: the caller supplies rows that
 * are zero (vings_surfel_project_launch_activate can clear them) or hold gradients to add to. */
int vings_surfel_blend_backward_accumulate(int N, int H, int W, const uint32_t* ranges,
                                const uint32_t* vals_sorted, const float* geom, const float* bg,
                                const uint8_t* pixel_mask, const float* final_T,
                                const uint32_t* n_contrib, const float* dL_dcolor,
                                const float* dL_dallmap, float* dgeom, void* stream);

/* ------------------------------------------------------------------------
 * Backward of stage 1: chains dgeom to the rasteriser inputs.
 * out: dL_dmeans3D[N,3] dL_dscales[N,2] dL_drotations[N,4] dL_dopacities[N]
 *      dL_dcolors[N,3]; optional dL_dmeans2D[N,3] (screen-space gradient,
 *      z = 0) and scores_grad[N,2] (gaussian_base.py:387) may be NULL.
 */
int vings_surfel_project_backward(int N, int H, int W, float scale_modifier,
                                  const float* means3D, const float* scales,
                                  const float* rotations, const float* viewmatrix,
                                  const float* projmatrix, const int32_t* radii,
                                  const float* dgeom, float* dL_dmeans3D, float* dL_dscales,
                                  float* dL_drotations, float* dL_dopacities, float* dL_dcolors,
                                  float* dL_dmeans2D, float* scores_grad, void* stream);

/* ------------------------------------------------------------------------
 * Row-masked Adam without bias correction:
 *   m = b1 m + (1-b1) g; v = b2 v + (1-b2) g^2; p -= lr m / (sqrt(v)+eps)
 * applied only to rows i with visible[i] != 0.  Serves
 * SparseGaussianAdam.step (gaussian_base.py:62,402).  `param` is [N,M].
 */
int vings_sparse_adam(float* param, const float* grad, float* exp_avg, float* exp_avg_sq,
                      const uint8_t* visible, float lr, float b1, float b2, float eps, int N,
                      int M, void* stream);

/* Same update for up to 8 parameter groups sharing one visibility mask in a
 * single launch (the five splat groups of gaussian_base.py:55-61). The
 * pointer/size arrays live in HOST memory; the device arrays they name must be 16-byte
 * aligned.  Invisible rows keep their values (a row sharing a 16-byte quad with a visible
 * row is written back unchanged). */
int vings_sparse_adam_multi(int n_groups, float* const* params_host,
                            const float* const* grads_host, float* const* exp_avgs_host,
                            float* const* exp_avg_sqs_host, const int* widths_host,
                            const float* lrs_host, const uint8_t* visible, float b1, float b2,
                            float eps, int N, void* stream);

/* The same update on gradients clipped by their global norm:
 *   norm = sqrt(sum over all groups and visible rows of g^2)
 *   g' = g * min(1, max_norm / (norm + 1e-6)), then the update above on g'
 * Gradients of invisible rows count in nothing; invisible rows keep their values (as above, one
 * that shares a 16-byte quad with a visible row is written back unchanged).  A norm
 * that is infinite or NaN skips the step on the device: parameters and moments stay.  The
 * factors 1-b1 and 1-b2 are formed in 64 bits (vings_sparse_adam* form them in float32).  `norm`
 * (device, one float) receives the norm before clipping, and infinity for a step that the guard
 * drops: a step was skipped exactly if its norm is not finite.  Up to 64 groups, each
 * with its own b1, b2 and eps; arrays need 4-byte alignment only.  `instance_count` (may be
 * NULL) and `capacity`: as in vings_sparse_adam_multi_guarded.  The workspace holds the partial
 * sums of the norm; nothing in it outlives the call. */
size_t vings_sparse_adam_clipped_workspace_bytes(int n_groups);
int vings_sparse_adam_clipped(int n_groups, float* const* params_host, const float* const* grads_host,
                              float* const* exp_avgs_host, float* const* exp_avg_sqs_host,
                              const int* widths_host, const float* lrs_host, const double* b1s_host,
                              const double* b2s_host, const float* epss_host, const uint8_t* visible,
                              int N, float max_norm, float* norm, void* workspace,
                              size_t workspace_bytes, const uint32_t* instance_count,
                              uint32_t capacity, void* stream);

/* ------------------------------------------------------------------------
 * Element types of the entry points that take more than float32. */
#define VINGS_F32 0
#define VINGS_BF16 1
#define VINGS_F16 2

/* ------------------------------------------------------------------------
 * Global norm of many gradient tensors, and clipping by it (the reference limits the gradients
 * of its tracker network between backward and the optimiser, frontend/modules/clipping.py).
 *   norm_kind 0: norm = sqrt(sum of squares over all tensors), 1: the largest magnitude
 *   clip: out = g * min(1, max_norm / (norm + 1e-6)), rounded once to the type of out
 * The lists live in HOST memory and are read before the call returns; tensors may be empty, of
 * different types and aligned to their element only.  Any number of tensors; sums are held in
 * 64 bits and joined in a fixed order.  `norm`: one float on the device, written in every case
 * (0 for empty lists); a NaN among the gradients gives a NaN norm, and NaN clipped gradients;
 * an infinity gives an infinite norm and the coefficient 0.
 * vings_grad_clip: outs[i] is grads[i] itself (in place; nothing is written when the coefficient
 * is 1) or memory that overlaps no other tensor of the call; its type is grads[i]'s or float32. */
size_t vings_grad_norm_workspace_bytes(int n_tensors, const int64_t* numels_host);
int vings_grad_norm(int n_tensors, const void* const* grads_host, const int64_t* numels_host,
                    const int* types_host, int norm_kind, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);
int vings_grad_clip(int n_tensors, const void* const* grads_host, void* const* outs_host,
                    const int64_t* numels_host, const int* types_host, const int* out_types_host,
                    int norm_kind, float max_norm, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Rows of a table by id, scaled, and the gradient of the table by sorted ids.
 *   vings_row_lookup            out[n] = scale * table[ids[n]], zeros where ids[n] is outside
 *                               [0, n_rows)
 *   vings_row_lookup_backward   rows[v] = scale * sum over {n : ids[n] == v} of grad[n]; rows[v]
 *                               of an id that does not occur is zero.  Ids outside [0, n_rows)
 *                               and ids equal to padding_id (-1: none) contribute nothing.
 * table / grad: row-major with table_stride / grad_stride elements between rows (grad_stride 0:
 * one row for all ids), of type VINGS_F32 / BF16 / F16; out, rows dense.  rows_type is the
 * gradient's type or VINGS_F32.  ids int32 or int64 (id_bytes).  Sums are float32, in an order
 * fixed by the ids alone, rounded once.  touched (may be NULL) [n_rows]: 1 for rows that some id
 * names, else 0 -- or left as it is with keep_touched, so that several calls can mark one array.
 * Sizes: n_ids, n_rows < 2^31 - 1, 0 < n_cols <= 2^20, grad_stride <= 2^20.  rows and touched
 * overlap no other array of the call. */
int vings_row_lookup(int64_t n_ids, int64_t n_rows, int64_t n_cols, const void* table,
                     int64_t table_stride, int type, const void* ids, int id_bytes, float scale,
                     void* out, void* stream);
size_t vings_row_lookup_backward_workspace_bytes(int64_t n_ids, int64_t n_rows, int64_t n_cols,
                                                 int type);
int vings_row_lookup_backward(int64_t n_ids, int64_t n_rows, int64_t n_cols, const void* grad,
                              int64_t grad_stride, int type, const void* ids, int id_bytes,
                              int64_t padding_id, float scale, void* rows, int rows_type,
                              uint8_t* touched, int keep_touched, void* workspace,
                              size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Parameter activations of get_property (gaussian_base.py:44-48,64-72):
 * opacity = sigmoid(raw), scaling = exp(raw), rotation = raw / max(|raw|, 1e-12)
 * (xyz and rgb are used as stored).  One launch for the three groups.
 */
int vings_splat_activate(int N, const float* raw_opacity, const float* raw_scaling,
                         const float* raw_rotation, float* opacities, float* scales,
                         float* rotations, void* stream);

/* After the rasteriser backward of one view, in one launch per splat:
 *  - chain rule through the activations above (gradients w.r.t. the stored parameters),
 *  - weighting_grad (gaussian_utils.py:56-62): every gradient row times
 *    s0 / (S0 + 1e-6 + s0), s0 = cur_scores[:,0], S0 = clamp(global_scores[:,0] + s0, 0, 1e4),
 *  - visible = radii > 0 && !stable_mask (the mask SparseGaussianAdam.step gets at
 *    gaussian_base.py:402; stable_mask may be NULL),
 *  - if bookkeeping != 0, add_records (gaussian_model.py:163-168): global_scores[:,0] = S0,
 *    local_scores[:,0] += s0, local_scores[:,1] = max(., cur_scores[:,1]), and the
 *    best-keyframe record (kf_max_scores, kf_id) takes (s0, this_kf) where s0 is larger.
 *    With several GPUs the caller reduces scores across ranks first and passes 0.
 * d_* are gradients w.r.t. the ACTIVATED values as vings_surfel_project_backward returns
 * them; g_* receive the weighted gradients w.r.t. the stored parameters (overwritten).
 */
int vings_splat_grad_finish(int N, const float* opacities, const float* scales,
                            const float* raw_rotation, const float* d_means3D,
                            const float* d_colors, const float* d_opacities, const float* d_scales,
                            const float* d_rotations, const float* cur_scores, const int* radii,
                            const uint8_t* stable_mask, float* global_scores, float* local_scores,
                            float* kf_max_scores, int64_t* kf_id, int64_t this_kf, int bookkeeping,
                            float* g_xyz, float* g_rgb, float* g_opacity, float* g_scaling,
                            float* g_rotation, uint8_t* visible, void* stream);

/* vings_surfel_project_backward and vings_splat_grad_finish in one launch, for the mapper's view
 * step (gaussian_base.py:385-403 straight after the rasteriser backward of
 * rasterize_points.cu / backward.cu preprocess): the gradients w.r.t. the activated
 * parameters stay in registers.  scales / rotations / opacities are the ACTIVATED values the
 * forward pass was given, raw_rotation the stored quaternion; the g_* and visible outputs
 * and the bookkeeping are exactly those of vings_splat_grad_finish (bit-identical).
 * scores_grad [N,2] (optional) receives the view's two scores as the unfused call does.
 * Multi-GPU form: with packed != NULL (then bookkeeping must be 0 and record_keys given) the
 * weighted gradients, s0 and the visibility flag go straight into the planar exchange buffer
 * and the record keys are folded into record_keys, exactly as vings_splat_pack_exchange would
 * do after this call; g_* and visible are then not written and may be NULL. */
int vings_surfel_project_backward_finish(
    int N, int H, int W, float scale_modifier, const float* means3D, const float* scales,
    const float* rotations, const float* viewmatrix, const float* projmatrix, const int32_t* radii,
    const float* dgeom, const float* opacities, const float* raw_rotation,
    const uint8_t* stable_mask, float* global_scores, float* local_scores, float* kf_max_scores,
    int64_t* kf_id, int64_t this_kf, int bookkeeping, float* g_xyz, float* g_rgb, float* g_opacity,
    float* g_scaling, float* g_rotation, uint8_t* visible, float* scores_grad, float* packed,
    int64_t* record_keys, void* stream);

/* ------------------------------------------------------------------------
 * Blend passes of the mapper's own view step.  Its loss (loss_utils.py:110-153 as called at
 * gaussian_base.py:367-382) has no term in the median depth nor in the blended flow, and the
 * mapper attaches no flow to its splats, so dL/dallmap[5], [7], [8] are identically zero.
 * The lean forward writes zeros into those three planes and 0 as the median's contributor
 * index, the lean backward does not read those three gradient planes, and neither does the
 * per-pair work behind them; every other output has the bits of the full passes.  Arguments as
 * vings_surfel_blend_forward / vings_surfel_blend_backward_accumulate.  Not for callers that
 * consume the median depth or the flow (the drop-in GaussianRasterizer uses the full passes). */
int vings_surfel_blend_forward_lean(int H, int W, const uint32_t* ranges,
                                    const uint32_t* vals_sorted, const float* geom,
                                    const float* bg, const uint8_t* pixel_mask, float* out_color,
                                    float* allmap, float* final_T, uint32_t* n_contrib,
                                    void* stream);
int vings_surfel_blend_backward_accumulate_lean(
    int N, int H, int W, const uint32_t* ranges, const uint32_t* vals_sorted, const float* geom,
    const float* bg, const uint8_t* pixel_mask, const float* final_T, const uint32_t* n_contrib,
    const float* dL_dcolor, const float* dL_dallmap, float* dgeom, void* stream);

/* Tile scheduling of the blend passes (no counterpart in the reference: its CUDA grid takes the
 * tiles in image order).  vings_surfel_tile_order writes a permutation of the T = ceil(W/16) *
 * ceil(H/16) tiles, longest list first (256 length classes; the order inside a class is
 * arbitrary), from the ranges vings_surfel_bin left.  The _ordered blend passes take their tiles
 * in that order (workgroup b renders tile tile_order[b]; NULL = the default XCD-contiguous
 * order), so a launch ends on its cheapest tiles and the workgroups dealt round-robin over the
 * XCDs carry similar loads.  Outputs have the bits of the unordered passes (the gradient rows up
 * to the order of their float atomics, as before; vings_surfel_blend_importance_ordered is
 * vings_surfel_blend_importance with that argument).  `lean` != 0 selects the lean passes above;
 * the backward adds into dgeom like vings_surfel_blend_backward_accumulate.  tile_order must be
 * a permutation of 0..T-1: a tile missing from it is not rendered. */
int vings_surfel_tile_order(int H, int W, const uint32_t* ranges, uint32_t* tile_order,
                            void* stream);
int vings_surfel_blend_forward_ordered(int lean, int H, int W, const uint32_t* ranges,
                                       const uint32_t* vals_sorted, const float* geom,
                                       const float* bg, const uint8_t* pixel_mask,
                                       float* out_color, float* allmap, float* final_T,
                                       uint32_t* n_contrib, const uint32_t* tile_order,
                                       void* stream);
int vings_surfel_blend_backward_accumulate_ordered(
    int lean, int N, int H, int W, const uint32_t* ranges, const uint32_t* vals_sorted,
    const float* geom, const float* bg, const uint8_t* pixel_mask, const float* final_T,
    const uint32_t* n_contrib, const float* dL_dcolor, const float* dL_dallmap, float* dgeom,
    const uint32_t* tile_order, void* stream);
/* The same backward pass for a map with splats the optimiser will not step: stable_mask[N]
 * (uint8, the mapper's _stable_mask; gaussian_base.py:400-402 zeroes their radii before
 * SparseGaussianAdam.step(radii > 0, N), so their gradients are never read, while
 * gaussian_model.py:163-168 records their scores like everybody's).  A flagged splat keeps its
 * place in the compositing of the pixels behind it and its two score sums (components 18, 19 of
 * its dgeom row); components 0..17 of its row stay as the caller cleared them.  Rows of
 * unflagged splats are what vings_surfel_blend_backward_accumulate_ordered leaves, up to the
 * order of the float atomics.  tile_order may be NULL; stable_mask NULL = no splat flagged.
 * vings_surfel_project_backward_finish given the same mask turns a flagged row into zero
 * gradients + recorded scores without reading components 0..17. */
int vings_surfel_blend_backward_accumulate_stable(
    int lean, int N, int H, int W, const uint32_t* ranges, const uint32_t* vals_sorted,
    const float* geom, const float* bg, const uint8_t* pixel_mask, const float* final_T,
    const uint32_t* n_contrib, const float* dL_dcolor, const float* dL_dallmap, float* dgeom,
    const uint32_t* tile_order, const uint8_t* stable_mask, void* stream);
/* The backward pass for a caller that does not know what its upstream gradient holds (the
 * autograd wrapper of GaussianRasterizer, gaussian_base.py:382): for splats WITHOUT flow
 * (u2_minus_u1 absent: the flow planes of dL_dallmap then multiply zeros) the lean pass is the
 * full pass whenever dL_dallmap[5] (median depth) is identically zero, which is what every loss
 * of the reference gives (loss_utils.py:110-153 has no term in it).  One small launch tests that
 * plane into flag_word (a caller-owned device word), then the lean and the full pass are both
 * launched and the one the flag does not select returns at its first instruction.  Adds into
 * dgeom like vings_surfel_blend_backward_accumulate_ordered; tile_order may be NULL.  Do not use
 * it with flow attached to the splats. */
int vings_surfel_blend_backward_auto(
    int N, int H, int W, const uint32_t* ranges, const uint32_t* vals_sorted, const float* geom,
    const float* bg, const uint8_t* pixel_mask, const float* final_T, const uint32_t* n_contrib,
    const float* dL_dcolor, const float* dL_dallmap, float* dgeom, const uint32_t* tile_order,
    uint32_t* flag_word, void* stream);
int vings_surfel_blend_importance_ordered(int N, int H, int W, const uint32_t* ranges,
                                          const uint32_t* vals_sorted, const float* geom,
                                          const uint8_t* pixel_mask, float* importance,
                                          int accumulate, const float* bg, float* rgb_max,
                                          const uint32_t* tile_order, void* stream);

/* ------------------------------------------------------------------------
 * The view step under HIP stream capture (one graph per keyframe of the window, replayed every
 * iteration).  A graph has fixed buffers, so the view is binned into a fixed capacity, and the
 * host cannot look at the instance count in the middle of it.  Three entry points make that
 * safe; none of them synchronises, records an event or touches the library's mailboxes:
 *   vings_surfel_project_enqueue_activate   vings_surfel_project_launch_activate with the three
 *       count words {depth bits min, max, instance count D} written to count_words, memory of
 *       the caller that the GPU can write (pinned host memory: the host reads D from it
 *       whenever it next looks; or device memory).  Follow it with
 *       vings_surfel_bin_speculative(capacity, tail = block_prefix + 3*ceil(N/256) + 1).
 *   vings_surfel_project_backward_finish_guarded, vings_sparse_adam_multi_guarded   the
 *       single-GPU finish (bookkeeping on) and the Adam step, which do NOTHING when
 *       *instance_count > capacity: a view whose instance list did not fit was blended from a
 *       truncated list, so its step is dropped as a whole and the map stays as it was; the
 *       caller sees D > capacity in count_words afterwards and repeats the step with room.
 * No counterpart in the reference (its view step is eager PyTorch, gaussian_base.py:353-404). */
int vings_surfel_project_enqueue_activate(
    int N, int H, int W, float scale_modifier, const float* means3D, const float* raw_scaling,
    const float* raw_rotation, const float* raw_opacity, const float* colors, const float* flow,
    const float* viewmatrix, const float* projmatrix, float* scales, float* rotations,
    float* opacities, float* geom, float* depth, int32_t* radii, int32_t* rect,
    uint32_t* tiles_touched, uint32_t* block_prefix, float* dgeom_clear, uint32_t* count_words,
    void* stream);
int vings_surfel_project_backward_finish_guarded(
    int N, int H, int W, float scale_modifier, const float* means3D, const float* scales,
    const float* rotations, const float* viewmatrix, const float* projmatrix, const int32_t* radii,
    const float* dgeom, const float* opacities, const float* raw_rotation,
    const uint8_t* stable_mask, float* global_scores, float* local_scores, float* kf_max_scores,
    int64_t* kf_id, int64_t this_kf, float* g_xyz, float* g_rgb, float* g_opacity,
    float* g_scaling, float* g_rotation, uint8_t* visible, const uint32_t* instance_count,
    uint32_t capacity, void* stream);
int vings_sparse_adam_multi_guarded(int n_groups, float* const* params_host,
                                    const float* const* grads_host, float* const* exp_avgs_host,
                                    float* const* exp_avg_sqs_host, const int* widths_host,
                                    const float* lrs_host, const uint8_t* visible, float b1,
                                    float b2, float eps, int N, const uint32_t* instance_count,
                                    uint32_t capacity, void* stream);

/* ------------------------------------------------------------------------
 * Compact exchange of one view step between the GPUs of a sharded mapping job (one process
 * per GPU, every GPU holds the whole splat set and renders its own keyframe; the reference is
 * single-GPU, configs/hierarchical/smallcity.yaml:11-13, so these have no counterpart there).
 * Only the rows some rank touched travel, in chunks that are reduced and applied one after
 * the other:
 *   1. vings_splat_touched          touched[i] = radii[i] > 0  (then MAX over the ranks)
 *   2. vings_splat_compact_plan_device  slot_of_row from the reduced mask; the slot count M
 *      goes to a DEVICE word (no read-back, no synchronisation; same dst_index as
 *      vings_splat_compact_plan)
 *   3. vings_surfel_project_backward_pack  the per-splat backward of the view with the weighted
 *      gradients and s0 written into the chunked buffer: slot s is in chunk c = s / chunk_rows,
 *      packed[(c*14 + column)*chunk_rows + (s - c*chunk_rows)], columns {g_xyz 3, g_rgb 3,
 *      g_opacity 1, g_scaling 2, g_rotation 4, s0}; rows_of_slot[s] = row; record keys folded
 *      as in vings_surfel_project_backward_finish.  packed must hold
 *      14 * chunk_rows * ceil(M / chunk_rows) floats.
 *   4. per chunk, after its SUM all-reduce: vings_splat_exchange_step(n_slots of the chunk,
 *      chunk_rows, chunk, rows_of_slot + first slot of the chunk, ...) adds the summed s0 to
 *      global_scores[:,0] (clamped to [0,1e4]) and local_scores[:,0] and applies the
 *      row-masked Adam update of vings_sparse_adam to the 13 parameters of every slot whose
 *      splat is not stable (params / exp_avgs / exp_avg_sqs / lrs: HOST arrays of 5 entries
 *      in the order xyz, rgb, opacity, scaling, rotation).
 */
int vings_splat_exchange_columns(void);
int vings_splat_touched(int N, const int32_t* radii, uint8_t* touched, void* stream);
int vings_splat_compact_plan_device(int N, const uint8_t* keep, int32_t* dst_index,
                                    void* workspace, size_t workspace_bytes,
                                    int64_t* n_keep_device, void* stream);
int vings_surfel_project_backward_pack(
    int N, int H, int W, float scale_modifier, const float* means3D, const float* scales,
    const float* rotations, const float* viewmatrix, const float* projmatrix, const int32_t* radii,
    const float* dgeom, const float* opacities, const float* raw_rotation,
    const float* global_scores, int64_t this_kf, float* scores_grad, float* packed,
    int64_t* record_keys, const int32_t* slot_of_row, int32_t* rows_of_slot, int chunk_rows,
    void* stream);
int vings_splat_exchange_step(int n_slots, int chunk_rows, const float* chunk,
                              const int32_t* rows, float* const* params_host,
                              float* const* exp_avgs_host, float* const* exp_avg_sqs_host,
                              const float* lrs_host, float b1, float b2, float eps,
                              const uint8_t* stable_mask, float* global_scores,
                              float* local_scores, void* stream);

/* ------------------------------------------------------------------------
 * Forward-only importance of every splat in one view: importance[i] (+)= sum over pixels of
 * the blend weight alpha*T, i.e. the value the backward pass leaves in scores.grad[:,0]
 * (it does not depend on the upstream gradient).  Serves the scoring passes that the
 * reference runs as render + backward of a throw-away loss: storage_control
 * (gaussian_model.py:233-241) and calc_score_v1 (loop/loop_model.py:169-214).  Takes the
 * outputs of vings_surfel_project / vings_surfel_bin; writes no image.
 * accumulate = 0 zeroes importance[N] first.  rgb_max (device float, may be NULL; needs bg[3])
 * receives max(0, largest value of the colour image this view would render), which
 * calc_score_v1 tests against 0.1 to skip empty views (loop_model.py:181).
 */
int vings_surfel_blend_importance(int N, int H, int W, const uint32_t* ranges,
                                  const uint32_t* vals_sorted, const float* geom,
                                  const uint8_t* pixel_mask, float* importance, int accumulate,
                                  const float* bg, float* rgb_max, void* stream);

/* ------------------------------------------------------------------------
 * Pruning: order-preserving compaction of every per-splat array by a keep mask, in place of
 * the array-by-array boolean indexing of prune_tensors_from_optimizer
 * (gaussian_base.py:94-110) and update_records(mode="prune") (gaussian_model.py:178-183).
 * plan : dst_index[i] = new row of splat i, or -1 if keep[i] == 0; *n_keep_host = rows kept
 *        (synchronises once to return it: the caller sizes the destination arrays with it).
 * apply: copies row i of each of the n_arrays source arrays (row_bytes_host[a] bytes per
 *        row; pointer tables in HOST memory, at most 24 arrays) to row dst_index[i] of the
 *        matching destination array.  Out of place.
 */
size_t vings_splat_compact_workspace_bytes(int N);
int vings_splat_compact_plan(int N, const uint8_t* keep, int32_t* dst_index, void* workspace,
                             size_t workspace_bytes, int64_t* n_keep_host, void* stream);
int vings_splat_compact_apply(int N, const int32_t* dst_index, int n_arrays,
                              const void* const* src_host, void* const* dst_host,
                              const int* row_bytes_host, void* stream);

/* The plan step for callers that cannot allocate (code under HIP graph capture, serving loops,
 * harnesses that forbid hipMalloc): no workspace argument, no host read-back, no
 * synchronisation.  It has no counterpart in the reference.  The per-block counts live in a
 * static device array of the library (128 KiB per GPU, held until the process ends), so N is
 * limited to vings_splat_compact_static_max_rows() = 8 388 608; a larger N is rejected with
 * VINGS_ERR_ARG.  The number of kept rows is written to the DEVICE word n_keep_device on the
 * stream.  dst_index is what vings_splat_compact_plan produces.  All calls on one GPU share
 * that GPU's scratch array: calls that overlap in time on one GPU (two streams, two threads)
 * race; calls on one stream do not.
 * The first call on a GPU looks up the address of that GPU's array (hipGetSymbolAddress, not a
 * stream operation).  A caller that records the call into a HIP graph does that lookup before
 * the capture begins with vings_splat_compact_static_prepare() (current device; idempotent;
 * allocates nothing) or with one ordinary call. */
int vings_splat_compact_static_max_rows(void);
int vings_splat_compact_static_prepare(void);
int vings_splat_compact_plan_static(int N, const uint8_t* keep, int32_t* dst_index,
                                    int64_t* n_keep_device, void* stream);

/* ------------------------------------------------------------------------
 * mean_dist2[i] = mean of the squared distances from point i to its three nearest other
 * points; xyz[N,3].  Serves distCUDA2 (gaussian_utils.py:12-16; callers gaussian_model.py:72,
 * 139: initial scale of new splats), which the reference runs as a k-d tree on the host.
 * N >= 4.
 */
int vings_knn3_mean_dist2(int N, const float* xyz, float* mean_dist2, void* stream);

/* World position and colour of n chosen pixels of a new keyframe (get_pointcloud,
 * gaussian_utils.py:39-46 with tf.py:46-68): pixel_ids[n] are row-major indices into
 * depth[H,W] / rgb[3,H,W]; pixel (row u, column v) of depth z maps to the camera point
 * ((v-cv)/fv*z, (u-cu)/fu*z, z) and through c2w_host (16 host floats, row major).
 * Writes xyz[n,3], colors[n,3]. */
int vings_keyframe_backproject(int n, int H, int W, const int64_t* pixel_ids, const float* depth,
                               const float* rgb, const float* c2w_host, float fu, float fv,
                               float cu, float cv, float* xyz, float* colors, void* stream);

/* ------------------------------------------------------------------------
 * Loop closure, per-splat stages.
 * top3_update: folds the importance of one more keyframe view into every splat's record of
 *   its three best keyframes, scores3[N,3] (descending) and kfids3[N,3] (int32), with the
 *   comparisons of calc_score_v1 (loop/loop_model.py:190-211; strict, so ties insert nothing).
 * reanchor: for every splat whose owning keyframe owner_kf[i*owner_stride] lies in
 *   [kf_start, kf_end]: xyz <- new_c2w[kf] * (scale[kf] * (old_w2c[kf] * xyz)), rotation <-
 *   delta_quat[kf] * rotation / |rotation| (loop/loop_rectify.py:322-367), in place.
 *   Pose tables are device arrays indexed by keyframe: old_w2c, new_c2w [K,12] (3x4 row
 *   major), delta_quat [K,4] (w,x,y,z; the rotation of new_c2w * old_w2c), scale [K].
 *   Quaternions are (w,x,y,z) throughout, as the rasteriser reads them; the reference
 *   round-trips this step through (x,y,z,w) libraries -- flagged, not reproduced.
 * depth_refresh: the tracker-side refresh after a loop closure (rectify_tracker,
 *   loop/loop_rectify.py:420-426) from the two rasteriser channels depth_sum[H,W] and
 *   alpha[H,W]: d = depth_sum/alpha with NaN and +inf -> 0 (gaussian_base.py:205-209);
 *   dense_map[H,W] takes d wherever d > 0 (in place, other pixels keep their value);
 *   coarse_map[H/8,W/8] = mean of the four centre pixels (rows/columns 3,4) of every 8x8
 *   block of the updated dense_map.  H and W must be multiples of 8.
 */
int vings_depth_refresh(int H, int W, const float* depth_sum, const float* alpha,
                        float* dense_map, float* coarse_map, void* stream);
int vings_splat_top3_update(int N, const float* cur_importance, int kf_id, float* scores3,
                            int32_t* kfids3, void* stream);
/* The same, skipped as a whole on the device when *gate < gate_min: the reference drops a view
 * whose render stays below 0.1 everywhere with a host-side test (loop/loop_model.py:181); with
 * gate = the rgb_max word of vings_surfel_blend_importance the host never waits for it. */
int vings_splat_top3_update_gated(int N, const float* cur_importance, int kf_id, float* scores3,
                                  int32_t* kfids3, const float* gate, float gate_min,
                                  void* stream);
/* Multi-GPU form of the scoring: the keyframe sequence of loop/loop_model.py:174 is dealt out
 * over R ranks in contiguous blocks (rank 0 the earliest keyframes), every rank builds its
 * record over its block with vings_splat_top3_update*, the records are gathered
 * (scores_all, kfids_all: [R,N,3], rank-major) and merged here.  The entries of rank r's
 * record pass through the same strict comparisons (loop_model.py:190-211), best first, ranks
 * in order: equal scores keep the earlier keyframe and empty slots (score 0) never enter, so
 * scores3 / kfids3 [N,3] equal what one pass over all keyframes leaves, bit for bit.  The
 * outputs must not alias the inputs. */
int vings_splat_top3_merge(int N, int R, const float* scores_all, const int32_t* kfids_all,
                           float* scores3, int32_t* kfids3, void* stream);
int vings_splat_reanchor(int N, float* xyz, float* rotation, const int32_t* owner_kf,
                         int owner_stride, int kf_start, int kf_end, int K, const float* old_w2c,
                         const float* new_c2w, const float* delta_quat, const float* scale,
                         void* stream);

/* Exchange between GPU replicas of the splat set (no counterpart in the reference, which is
 * single-GPU: configs/hierarchical/smallcity.yaml:11-13).  After vings_splat_grad_finish with
 * bookkeeping = 0, pack writes vings_splat_pack_columns() = 15 planar columns of N floats
 * {g_xyz 3, g_rgb 3, g_opacity, g_scaling 2, g_rotation 4, s0, visible} (packed[c*N + i]) to
 * be SUMMED over ranks after every view; unpack takes the summed buffer back into the
 * gradient arrays and the visibility mask and adds the summed s0 to the score records
 * (add_records, gaussian_model.py:163-168).  The two record maxima that no view step reads
 * (best keyframe per splat, error score) are not exchanged per view: pack folds
 * {bits(max(s0,0)) << 32 | this_kf, bits(max(s1,0))} into the running maximum held in
 * record_keys [N,2] (zero it once); when the records are needed the caller MAXIMISES
 * record_keys over ranks and vings_splat_merge_records folds it into local_scores[:,1],
 * kf_max_scores and kf_id and zeroes it again. */
int vings_splat_pack_columns(void);
int vings_splat_pack_exchange(int N, const float* g_xyz, const float* g_rgb,
                              const float* g_opacity, const float* g_scaling,
                              const float* g_rotation, const uint8_t* visible,
                              const float* cur_scores, int64_t this_kf, float* packed,
                              int64_t* record_keys, void* stream);
int vings_splat_unpack_exchange(int N, const float* packed, float* global_scores,
                                float* local_scores, float* g_xyz, float* g_rgb,
                                float* g_opacity, float* g_scaling, float* g_rotation,
                                uint8_t* visible, void* stream);
int vings_splat_merge_records(int N, int64_t* record_keys, float* local_scores,
                              float* kf_max_scores, int64_t* kf_id, void* stream);

/* ------------------------------------------------------------------------
 * Mapping loss of one rendered view and its gradient w.r.t. the rasteriser
 * outputs, in place of the PyTorch graph + autograd pass the reference builds
 * per view between GaussianRasterizer.forward and .backward:
 *   render post-processing  gaussian_base.py:205-224   (depth = A0/alpha with
 *                           nan/inf -> 0, normals to the world frame)
 *   depth -> normal         normal_utils.py:6-21       (central differences)
 *   get_loss, use_sky off   loss_utils.py:110-153      (0.8 L1 + 0.2 (1-SSIM),
 *                           normal, alpha-on-sky, depth / depth_cov, dist)
 *   ssim                    loss_utils.py:26-57        (11x11 Gaussian, sigma 1.5)
 * Device arrays: rgb [3,H,W], allmap [9,H,W] (rasteriser outputs), gt_rgb
 * [3,H,W], gt_depth [H,W], gt_depth_cov [H,W]; outputs dL_drgb [3,H,W],
 * dL_dallmap [9,H,W] (every element written), loss_out [8] = total, rgb,
 * normal, alpha, depth, dist terms, valid-pixel count, sky-pixel count.
 * HOST arrays: Rw2c [9] (row-major rotation of the world->camera matrix),
 * weights [5] = rgb, depth, alpha, normal, dist (training_args.loss_weights).
 * fu, cu belong to the row (vertical) axis, fv, cv to the column axis.
 * Empty masks divide by 1 instead of producing NaN.  Gradients of pixels whose
 * depth = A0/alpha is not finite are zero where autograd would give NaN.
 * Nothing synchronises with the host.
 */
size_t vings_mapping_loss_workspace_bytes(int H, int W);
int vings_mapping_loss(int H, int W, const float* rgb, const float* allmap, const float* gt_rgb,
                       const float* gt_depth, const float* gt_depth_cov, const float* Rw2c_host,
                       float fu, float fv, float cu, float cv, const float* weights_host,
                       float* dL_drgb, float* dL_dallmap, float* loss_out, void* workspace,
                       size_t workspace_bytes, void* stream);
/* The same with the parts that depend on the keyframe's ground truth alone kept between calls
 * (the mapper iterates over a keyframe many times, gaussian_base.py:353-404, while its images
 * stay what they are): the Gaussian-filtered mean and second moment of gt_rgb, the pixel
 * classes (valid / sky) and their counts.  gt_cache: vings_mapping_loss_gt_cache_bytes(H, W)
 * bytes of device memory owned by the caller, 8-byte aligned, one per keyframe.
 * gt_cache_valid = 0: computed as in vings_mapping_loss and stored; 1: read (the SSIM forward
 * pass then filters three moments instead of five).  Results are bit-identical to
 * vings_mapping_loss either way.  The caller resets the flag when it changes gt_rgb / gt_depth. */
size_t vings_mapping_loss_gt_cache_bytes(int H, int W);
int vings_mapping_loss_cached(int H, int W, const float* rgb, const float* allmap,
                              const float* gt_rgb, const float* gt_depth,
                              const float* gt_depth_cov, const float* Rw2c_host, float fu, float fv,
                              float cu, float cv, const float* weights_host, float* dL_drgb,
                              float* dL_dallmap, float* loss_out, void* workspace,
                              size_t workspace_bytes, void* gt_cache, int gt_cache_valid,
                              void* stream);

/* ========================================================================
 * Dense bundle adjustment (droid_backends).
 *
 * Shapes as passed by the reference (depth_video.py:380-381, 654-659):
 *   poses[B,7] (tx,ty,tz,qx,qy,qz,qw; world->camera)   disps[B,ht,wd]
 *   intr[4] = fx,fy,cx,cy at grid resolution             disps_sens[B,ht,wd] or NULL
 *   target, weight [E,2,ht,wd]   eta[M,ht,wd]   ii, jj [E] int64 (device)
 * Poses t0 <= f < t1 are free (P = t1-t0); the M depth variables are the
 * sorted unique of arange(t0,t1) and ii, so M equals the row count of eta.
 * All state between stages lives in one caller-provided workspace whose
 * layout is returned by vings_dba_layout_query (byte offsets).
 * ======================================================================== */
typedef struct vings_dba_layout {
    size_t total_bytes;
    size_t off_E;         /* double [(P+E),6,HW] coupling rows: P per-pose rows, then per edge */
    size_t off_Q;         /* double [M,HW] inverse of the depth block                     */
    size_t off_w;         /* double [M,HW] depth residual                                */
    size_t off_H;         /* double [8][6P,6P] undamped pose block as 8 partial sums, lower triangle only */
    size_t off_v;         /* double [8][6P] as 8 partial sums                            */
    size_t off_S;         /* double [8][6P,6P] Schur complement E Q E^T, like H          */
    size_t off_u;         /* double [8][6P] E Q w as 8 partial sums                      */
    size_t off_dx;        /* double [6P]    pose update                                  */
    size_t off_chol;      /* double [6P,6P] factorisation scratch                        */
    size_t off_kx;        /* int32  [M] frame of each depth variable                     */
    size_t off_kk;        /* int32  [E] depth variable of each edge                      */
    size_t off_kstart;    /* int32  [M+1] edge list offsets                              */
    size_t off_kedges;    /* int32  [E]                                                  */
    size_t off_ip;        /* int32  [E] ii                                               */
    size_t off_jp;        /* int32  [E] jj                                               */
    size_t off_ent_start; /* int32  [M+1] entry list offsets                             */
    size_t off_ent_row;   /* int32  [P+E] row block of E                                 */
    size_t off_ent_pose;  /* int32  [P+E] free-pose index of that row block              */
    size_t off_status;    /* int32  [4]: depth variables found, Cholesky failed, bad index */
} vings_dba_layout;

int vings_dba_layout_query(int ht, int wd, int E, int P, int M, vings_dba_layout* out);

/* droid_backends.ba (depth_video.py:380-381): `itrs` damped Gauss-Newton
 * iterations, poses[t0:t1] and disps updated IN PLACE.  Damping
 * H + (ep + lm*diag H) I, Schur elimination of the depth block, float64
 * Cholesky on the device; a failed factorisation leaves that iteration's
 * update at zero (chol.py:9-17). */
int vings_dba_ba(float* poses, float* disps, const float* intr, const float* disps_sens,
                 const float* target, const float* weight, const float* eta, const int64_t* ii,
                 const int64_t* jj, int B, int ht, int wd, int E, int M, int t0, int t1, int itrs,
                 float lm, float ep, int motion_only, void* workspace, size_t workspace_bytes,
                 void* stream);

/* BACore.init (depth_video.py:475-477,554): Jacobian stage + accumulation +
 * Schur complement, left in the workspace. */
int vings_dba_linearize(const float* poses, const float* disps, const float* intr,
                        const float* disps_sens, const float* target, const float* weight,
                        const float* eta, const int64_t* ii, const int64_t* jj, int B, int ht,
                        int wd, int E, int M, int t0, int t1, int motion_only, void* workspace,
                        size_t workspace_bytes, void* stream);

/* BACore.hessian (depth_video.py:478-481,550-551,618): reduced camera system
 * H_out[6P,6P] = H - S, v_out[6P] = v - u (float64, DEVICE buffers; the
 * Python mirror copies them into the caller's CPU tensors). */
int vings_dba_reduced_system(int B, int ht, int wd, int E, int M, int t0, int t1, void* workspace,
                             size_t workspace_bytes, double* H_out, double* v_out, void* stream);

/* BACore.hessian_expand (depth_video.py:568, consumed at 703-714): float32
 * copies Q_out[M,HW] and E_out[(P+E),6,HW] (first P row blocks = coupling of
 * each free pose with its own depth map, then one block per edge = coupling of
 * pose jj with the depth map of ii; blocks of fixed poses are zero). */
int vings_dba_export(int B, int ht, int wd, int E, int M, int t0, int t1, void* workspace,
                     size_t workspace_bytes, float* Q_out, float* E_out, void* stream);

/* BACore.retract (depth_video.py:649-650): applies pose update dx[6P]
 * (float64, device; NULL = use the update stored by the solver) and the
 * back-substituted depth update to poses / disps in place. */
int vings_dba_retract(float* poses, float* disps, const double* dx, int B, int ht, int wd, int E,
                      int M, int t0, int t1, int motion_only, void* workspace,
                      size_t workspace_bytes, void* stream);

/* droid_backends.frame_distance (depth_video.py:289-299): mean induced flow
 * magnitude per candidate edge, beta-weighted mix of full motion and
 * translation only; pairs with < 75 % valid weight return 1000. out[E]. */
int vings_frame_distance(const float* poses, const float* disps, const float* intr,
                         const int64_t* ii, const int64_t* jj, int B, int ht, int wd, int E,
                         float beta, float* out, void* stream);

/* droid_backends.corr_index_forward / _backward (modules/corr.py:12,19):
 * bilinear lookup of a (2r+1)^2 window around coords[E,2,h1,w1] in
 * volume[E,h1,w1,h2,w2] -> corr[E,2r+1,2r+1,h1,w1]; backward scatters
 * corr_grad into volume_grad (zeroed by the call).  half != 0: volume and
 * corr are float16 (the reference runs this under autocast).
 * Channel convention: corr[e,i,j,y,x] is the bilinear sample of volume[e,y,x,:,:] at
 * (coords.x + i - r, coords.y + j - r) -- the X offset is the SLOW index, the Y offset the fast
 * one, as in the public DROID-SLAM kernels the reference's extension descends from.  The
 * update operator's pretrained weights (droid.pth) convolve over these 4 * 49 channels
 * (modules/corr.py:46-50), so the order is part of the contract; the extension's source is not
 * in the reference tree, so the order is restated from that upstream layout, not pinned. */
int vings_corr_index_forward(const void* volume, const float* coords, void* corr, int E, int h1,
                             int w1, int h2, int w2, int r, int half, void* stream);
int vings_corr_index_backward(const float* coords, const void* corr_grad, void* volume_grad, int E,
                              int h1, int w1, int h2, int w2, int r, int half, void* stream);

/* droid_backends.altcorr_forward / altcorr_backward (modules/corr.py:79,86-87; operands built at
 * corr.py:106-125): the same window without the all-pairs volume.
 *   fmap1[B,H,W,C], fmap2[B,H2,W2,C] float32 (channels last, as corr.py:102 permutes them),
 *   coords[B,S,H,W,2] = (x, y) in fmap2 pixels, corr[B,S,(2r+1)^2,H,W].
 * corr[b,s,i*(2r+1)+j,h,w] = bilinear sample at (x + i - r, y + j - r) (X offset slow, the
 * channel convention of vings_corr_index_forward) of
 * (yy, xx) -> <fmap1[b,h,w,:], fmap2[b,yy,xx,:]>, zero outside fmap2: equal to
 * vings_corr_index_forward on volume = fmap1 . fmap2^T.  C a multiple of 4, <= 512; r <= 7.
 * backward: fmap1_grad, fmap2_grad (same shapes as the maps, zeroed by the call) receive the
 * adjoint of corr_grad[B,S,(2r+1)^2,H,W]; the gradient with respect to coords is not formed
 * (the host mirror returns zeros for the third element of the reference's 3-tuple). */
int vings_altcorr_forward(const float* fmap1, const float* fmap2, const float* coords, float* corr,
                          int B, int S, int H, int W, int H2, int W2, int C, int r, void* stream);
int vings_altcorr_backward(const float* fmap1, const float* fmap2, const float* coords,
                           const float* corr_grad, float* fmap1_grad, float* fmap2_grad, int B,
                           int S, int H, int W, int H2, int W2, int C, int r, void* stream);

/* ========================================================================
 * Tracker -> mapper packaging.
 * ======================================================================== */

/* compute_covariances (depth_video.py:676-726).  For depth variable k (frame kx[k]) and
 * pixel p:  e = the 6P coupling rows selected by block_of[K,P] (row block of E[(P+E),6,HW]
 * as vings_dba_export lays it out, -1 = zero block), F = (Q[k,p] e)^T L_inv with
 * L_inv[6P,6P] the inverse of the lower Cholesky factor of the reduced camera matrix
 * (row major, device), and depths_cov[kx[k],p] = (Q + |F|^2) / (disps[kx[k],p]^4 + 1e-6).
 * Q[K,HW]; disps, depths_cov [B,ht,wd]; kx[K] int64 (device).  P <= 20. */
int vings_depth_covariance(int ht, int wd, int P, int K, const float* Q, const float* E,
                           const int32_t* block_of, const float* L_inv, const float* disps,
                           const int64_t* kx, float* depths_cov, void* stream);

/* cvx_upsample (droid_net.py:17-38) as DepthVideo.upsample applies it (depth_video.py:236-243):
 * for the K frames ix[k] (int64, device) every coarse cell of src[f][B,ht,wd] becomes an 8x8
 * patch of dst[f][B,8ht,8wd], each output the softmax(mask[k, 0..8, i, j, y, x])-weighted sum
 * of the cell's 3x3 neighbourhood (zero padded); mask[K,576,ht,wd] float32, channel
 * (n*8+i)*8+j.  n_fields (1..4) maps share one pass over the mask; src_host / dst_host are
 * host arrays of device pointers; dst pointers 16-byte aligned. */
int vings_upsample_maps(int K, int ht, int wd, const int64_t* ix, const float* mask, int n_fields,
                        const float* const* src_host, float* const* dst_host, void* stream);

/* judge_and_package_v3, the array work (middleware_utils.py:224-238): for the n frames
 * frame_ids[n] (int64, device) of images[B,3,H,W] uint8, disps_up[B,H,W], depths_cov_up[B,H,W]:
 *   cov_median[f] = median of the frame's covariance map (mean of the two middle values for
 *                   an even count, like numpy.median);
 *   depths[n,H,W]  = 1/(disps_up+1e-6), 0 where that exceeds max_depth or the covariance
 *                   exceeds cov_times * cov_median[f];
 *   rgbs[n,H,W,3]  = images/255, 0 where depths == 0;
 *   depths_cov[n,H,W] = the covariance, replaced where depths == 0 by the largest covariance
 *                   of any pixel (all frames) that kept a positive depth (NaN if none did;
 *                   the reference raises there).
 * The maps must not hold NaN.  No host synchronisation. */
size_t vings_package_workspace_bytes(int n_frames);
int vings_package_keyframes(int n_frames, int H, int W, const int64_t* frame_ids,
                            const uint8_t* images, const float* disps_up,
                            const float* depths_cov_up, float max_depth, float cov_times,
                            float* rgbs, float* depths, float* depths_cov, float* cov_median,
                            void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Optional per-kernel timing with HIP events on the caller's stream (no
 * counterpart in the reference, whose only timers are the wandb brackets of
 * /root/reference/scripts/gaussian/wandb_utils.py:30-45).  enable(1) creates
 * an event pool once and resets the counters; read() synchronises on the
 * recorded events and returns the summed milliseconds / launch count of a tag.
 */
int vings_profile_enable(int on);
/* Restricts the timing to the tags whose bit is set (bit t = tag t; default all): every timed
 * launch costs two event records on the stream, a few microseconds each. */
int vings_profile_select(uint32_t tag_mask);
int vings_profile_num_tags(void);
const char* vings_profile_tag_name(int tag);
int vings_profile_read(int tag, double* total_ms, int64_t* count);

#ifdef __cplusplus
}
#endif
#endif /* VINGS_HIP_H */

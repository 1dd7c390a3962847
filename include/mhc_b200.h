/*
 * mhc_b200.h -- C-ABI of the B200 (sm_100a) mHC kernels.
 *
 * This is the drop-in boundary that replaces the reference's pybind11 module
 * `mhc_ascend` (ParadoxZW/mHC_Ascend, src/python/bindings.cpp:1020-1117).  Each
 * entry point below names the reference function it replaces.
 *
 * Conventions (all entry points):
 *   - Every pointer is a DEVICE pointer to contiguous row-major fp32 data
 *     (bf16 only where the name says so), on the device that is current for
 *     the calling thread.  `stream` is a cudaStream_t passed as void*.
 *   - Outputs are written, never accumulated into; the caller allocates them
 *     (the reference allocates fresh outputs with at::empty; here the Python
 *     layer allocates them with torch and passes them in).
 *   - Scalars that are parameters of the model (alpha, biases) are passed as
 *     device pointers, so a call never synchronises the host (the reference
 *     calls .item() on them: src/python/mhc/ops.py:420-422, 533-535).
 *   - Entry points that need scratch memory take (workspace, workspace_bytes)
 *     and have a *_workspace_bytes() query; they never allocate.
 *   - Return 0 (MHC_OK) on success, a negative MHC_ERR_* code otherwise;
 *     mhc_get_last_error_string() then describes the failure (per thread).
 *   - No entry point synchronises the stream or the device.
 */
#ifndef MHC_B200_H_
#define MHC_B200_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define MHC_API __attribute__((visibility("default")))
#else
#define MHC_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define MHC_OK 0
#define MHC_ERR_INVALID_ARG (-1)  /* bad shape / NULL pointer / bad hyper-parameter */
#define MHC_ERR_UNSUPPORTED (-2)  /* valid request this build does not implement */
#define MHC_ERR_ALIGNMENT (-3)    /* pointer not 16-byte aligned where required */
#define MHC_ERR_WORKSPACE (-4)    /* workspace NULL or smaller than *_workspace_bytes() */
#define MHC_ERR_CUDA (-5)         /* a CUDA launch reported an error */

/* Library identification and the per-thread description of the last error. */
MHC_API const char* mhc_version(void);
MHC_API const char* mhc_get_last_error_string(void);

/* ---------------------------------------------------------------------------
 * Sinkhorn-Knopp on a batch of square matrices [batch, n, n], 1 <= n <= 32.
 * Each iteration divides rows by (row sum + eps), then columns by
 * (column sum + eps) -- reference formulation ops_pytorch_backward.py:9-33.
 * ------------------------------------------------------------------------- */
/* replaces sinkhorn_knopp_fwd (bindings.cpp:155-187) */
MHC_API int mhc_sinkhorn_knopp_fwd(const float* inp, float* out, int64_t batch, int32_t n,
                           int32_t num_iters, float eps, void* stream);
/* replaces sinkhorn_knopp_bwd (bindings.cpp:189-231); exact reverse mode of
 * the forward above.  `out` (the forward result) is accepted for interface
 * parity and is not read: the forward is replayed from `inp`. */
MHC_API int mhc_sinkhorn_knopp_bwd(const float* grad_out, const float* inp, const float* out,
                           float* grad_inp, int64_t batch, int32_t n, int32_t num_iters,
                           float eps, void* stream);

/* ---------------------------------------------------------------------------
 * RMSNorm over rows of [batch, hidden]: out = inp / sqrt(mean(inp^2)+eps) * w
 * ------------------------------------------------------------------------- */
/* replaces rmsnorm_fwd (bindings.cpp:237-265); rms[batch] receives the row rms */
MHC_API int mhc_rmsnorm_fwd(const float* inp, const float* weight, float* out, float* rms,
                    int64_t batch, int64_t hidden, float eps, void* stream);
/* replaces rmsnorm_bwd (bindings.cpp:267-301).  grad_weight is a fixed-order
 * (atomic-free, deterministic) reduction over rows through the workspace. */
MHC_API size_t mhc_rmsnorm_bwd_workspace_bytes(int64_t batch, int64_t hidden);
MHC_API int mhc_rmsnorm_bwd(const float* grad_out, const float* inp, const float* weight,
                    const float* rms, float* grad_inp, float* grad_weight, int64_t batch,
                    int64_t hidden, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Stream aggregate: out[b,c] = sum_i sigmoid(H_pre_raw[b,i]) * inp[b,i,c]
 * ------------------------------------------------------------------------- */
/* replaces stream_aggregate_fwd (bindings.cpp:307-340); also writes
 * H_pre_act = sigmoid(H_pre_raw).  Output is fp32 (the reference writes bf16). */
MHC_API int mhc_stream_aggregate_fwd(const float* inp, const float* H_pre_raw, float* out,
                             float* H_pre_act, int64_t batch, int32_t n, int64_t hidden,
                             void* stream);
/* replaces stream_aggregate_bwd (bindings.cpp:342-374): grad_inp[b,i,c] =
 * H_pre_act[b,i]*grad_out[b,c]; grad_H_pre_act[b,i] = sum_c grad_out*inp. */
MHC_API int mhc_stream_aggregate_bwd(const float* grad_out, const float* inp, const float* H_pre_act,
                             float* grad_inp, float* grad_H_pre_act, int64_t batch, int32_t n,
                             int64_t hidden, void* stream);

/* ---------------------------------------------------------------------------
 * Stream distribute-mix-add:
 *   out[b,i,c] = 2*sigmoid(H_post_raw[b,i]) * y_norm[b,c] + sum_j M[b,i,j] x[b,j,c]
 * ------------------------------------------------------------------------- */
/* replaces stream_distribute_mix_add_fwd (bindings.cpp:380-412); also writes
 * H_post_act = 2*sigmoid(H_post_raw). */
MHC_API int mhc_stream_distribute_mix_add_fwd(const float* y_norm, const float* H_post_raw,
                                      const float* M, const float* x_inp, float* out,
                                      float* H_post_act, int64_t batch, int32_t n,
                                      int64_t hidden, void* stream);
/* replaces stream_distribute_mix_add_bwd (bindings.cpp:414-460): gradients
 * w.r.t. x, y_norm, M and H_post_act (the caller applies the activation
 * derivative, as ops.py:240-242 does). */
MHC_API int mhc_stream_distribute_mix_add_bwd(const float* grad_out, const float* x_inp,
                                      const float* y_norm, const float* M,
                                      const float* H_post_act, float* grad_x,
                                      float* grad_y_norm, float* grad_M,
                                      float* grad_H_post_act, int64_t batch, int32_t n,
                                      int64_t hidden, void* stream);

/* ---------------------------------------------------------------------------
 * Row RMS and the dynamic-H projection
 * ------------------------------------------------------------------------- */
/* replaces compute_rms_fwd (bindings.cpp:543-566): rms[b] = sqrt(mean(inp[b]^2)+eps) */
MHC_API int mhc_compute_rms_fwd(const float* inp, float* rms, int64_t batch, int64_t k, float eps,
                        void* stream);
/* replaces fused_rmsnorm_matmul_fwd (bindings.cpp:480-528): out[b,o] =
 * sum_k inp[b,k]*weight[o,k], computed in fp32 (the reference casts to bf16). */
MHC_API int mhc_fused_rmsnorm_matmul_fwd(const float* inp, const float* weight, float* out,
                                 int64_t batch, int64_t k, int32_t out_dim, void* stream);
/* replaces fused_rmsnorm_matmul_bwd (bindings.cpp:530-541): grad_inp =
 * grad_out @ weight, grad_weight = grad_out^T @ inp (fixed-order reduction). */
MHC_API size_t mhc_fused_rmsnorm_matmul_bwd_workspace_bytes(int64_t batch, int64_t k, int32_t out_dim);
MHC_API int mhc_fused_rmsnorm_matmul_bwd(const float* grad_out, const float* inp, const float* weight,
                                 float* grad_inp, float* grad_weight, int64_t batch, int64_t k,
                                 int32_t out_dim, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* ---------------------------------------------------------------------------
 * MHCResidualWrapper in one piece (replaces layer.py:287-316 around the fused
 * layer, bindings.cpp:600-952): for n = 4, fp32, hidden % 32 == 0 and 16-byte
 * aligned tensors, the streams are built inside the layer kernels from
 * residual / branch ([tokens, hidden] each; stream i = scales[i] * residual,
 * stream 1 = branch, exactly as mhc_wrapper_pack_fwd computes them) and the
 * forward writes the stream mean out_mean [tokens, hidden] -- the packed input
 * and the layer output never reach memory.  Workspaces and token_state as for
 * mhc_layer_fwd_dynamic / mhc_layer_bwd_dynamic with batch = tokens.  The
 * backward takes the mean's gradient and writes the residual and branch
 * gradients plus the parameter gradients (written, not accumulated).  Other
 * shapes return MHC_ERR_UNSUPPORTED (use the pack / layer / mean entry points).
 * ------------------------------------------------------------------------- */
MHC_API int mhc_wrapper_fwd_dynamic(const float* residual, const float* branch, const float* scales,
                                    const float* rmsnorm_weight, const float* phi_pre,
                                    const float* phi_post, const float* phi_res,
                                    const float* alpha_pre, const float* alpha_post,
                                    const float* alpha_res, const float* b_pre,
                                    const float* b_post, const float* b_res, float* out_mean,
                                    float* token_state, int64_t tokens, int32_t n, int64_t hidden,
                                    int32_t sinkhorn_iters, float sinkhorn_eps, float rmsnorm_eps,
                                    void* workspace, size_t workspace_bytes, void* stream);
/* The wrapper forward fused with the next branch's input RMSNorm (a pre-norm
 * block normalises the returned hidden state before its attention / MLP; the
 * reference composes MHCResidualWrapper.forward (layer.py:287-316) with the
 * branch's rmsnorm (ops.py:87-136) as two passes).  Writes out_mean as
 * mhc_wrapper_fwd_dynamic does, and out_normed[t, c] = out_mean[t, c] /
 * out_norm_rms[t] * norm_weight[c], out_norm_rms[t] = sqrt(mean_c out_mean^2
 * + norm_eps), from the same pass.  The backward of the norm is
 * mhc_rmsnorm_bwd on (grad_normed, out_mean, norm_weight, out_norm_rms); its
 * input gradient adds to grad_mean of mhc_wrapper_bwd_dynamic.  Same
 * requirements and workspace as mhc_wrapper_fwd_dynamic; norm_weight and
 * out_normed 16-byte aligned. */
MHC_API int mhc_wrapper_fwd_dynamic_prenorm(
    const float* residual, const float* branch, const float* scales, const float* rmsnorm_weight,
    const float* phi_pre, const float* phi_post, const float* phi_res, const float* alpha_pre,
    const float* alpha_post, const float* alpha_res, const float* b_pre, const float* b_post,
    const float* b_res, const float* norm_weight, float norm_eps, float* out_mean,
    float* out_normed, float* out_norm_rms, float* token_state, int64_t tokens, int32_t n,
    int64_t hidden, int32_t sinkhorn_iters, float sinkhorn_eps, float rmsnorm_eps,
    void* workspace, size_t workspace_bytes, void* stream);
MHC_API int mhc_wrapper_bwd_dynamic(const float* grad_mean, const float* residual,
                                    const float* branch, const float* scales,
                                    const float* rmsnorm_weight, const float* phi_pre,
                                    const float* phi_post, const float* phi_res,
                                    const float* alpha_pre, const float* alpha_post,
                                    const float* alpha_res, const float* b_pre,
                                    const float* b_post, const float* b_res,
                                    const float* token_state, float* grad_residual,
                                    float* grad_branch, float* grad_rmsnorm_weight,
                                    float* grad_phi_pre, float* grad_phi_post, float* grad_phi_res,
                                    float* grad_alpha_pre, float* grad_alpha_post,
                                    float* grad_alpha_res, float* grad_b_pre, float* grad_b_post,
                                    float* grad_b_res, int64_t tokens, int32_t n, int64_t hidden,
                                    int32_t sinkhorn_iters, float sinkhorn_eps, float rmsnorm_eps,
                                    void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * MHCResidualWrapper stream packing and stream mean (replace the framework ops
 * of layer.py:287-316; the reference has no native counterpart).  Tokens are
 * the flattened leading dims, x is [tokens, n, hidden] fp32, n <= 64.
 * scales: host array of n floats; stream i (i != 1) is scales[i] * residual
 * (scales[0] is taken as 1; "decay" mode passes 0.1^(i-1), "zero" mode 0, and
 * a zero scale writes 0).  Stream 1 is the branch output.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_wrapper_pack_fwd(const float* residual, const float* branch, float* out,
                                 const float* scales, int64_t tokens, int32_t n, int64_t hidden,
                                 void* stream);
/* bf16 residual / branch_output (tokens x hidden bf16, 8-byte aligned for the
 * vector path), fp32 streams out: the reference packs in residual.dtype
 * (layer.py:299-308), so streams i >= 2 are scales[i] * residual rounded to
 * bf16 before the layer widens them (layer.py:101). */
MHC_API int mhc_wrapper_pack_fwd_bf16(const void* residual, const void* branch, float* out,
                                      const float* scales, int64_t tokens, int32_t n,
                                      int64_t hidden, void* stream);
/* grad_residual = sum_{i != 1} scales[i] * grad[:, i]; grad_branch = grad[:, 1] (may be NULL) */
MHC_API int mhc_wrapper_pack_bwd(const float* grad_out, float* grad_residual, float* grad_branch,
                                 const float* scales, int64_t tokens, int32_t n, int64_t hidden,
                                 void* stream);
/* out[t, c] = mean_i inp[t, i, c]  (MHCResidualWrapper's output.mean(dim=1)) */
MHC_API int mhc_stream_mean_fwd(const float* inp, float* out, int64_t tokens, int32_t n,
                                int64_t hidden, void* stream);
/* grad_inp[t, i, c] = grad_out[t, c] / n */
MHC_API int mhc_stream_mean_bwd(const float* grad_out, float* grad_inp, int64_t tokens, int32_t n,
                                int64_t hidden, void* stream);

/* ---------------------------------------------------------------------------
 * Fused mHC layer, dynamic H.
 *
 * Per-token record saved by the forward for the backward ("token_state",
 * [batch, mhc_token_state_stride(n)] fp32):
 *   [0] rms_h  (rms of the flattened n*C token vector)
 *   [1] rms    (rms of the aggregated stream, RMSNorm denominator)
 *   [2, 2+n)          H_pre_act  = sigmoid(H_pre_tilde)
 *   [2+n, 2+2n)       H_post_act = 2*sigmoid(H_post_tilde)
 *   [2+2n, 2+2n+n*n)  M          = Sinkhorn(exp(H_res_tilde))
 *   [2+2n+n*n, ...+n*n+2n)  raw projections p = x_flat @ phi^T (pre|post|res)
 *   then, from the next even index, n(n+1)/2 doubles: the upper triangle of
 *   the token's Gram matrix x x^T (row-major), accumulated in fp64 from exact
 *   products; the record (and therefore the buffer) must be 8-byte aligned.
 *   Stride at n = 4: 72 floats.
 * ------------------------------------------------------------------------- */
MHC_API int32_t mhc_token_state_stride(int32_t n);

/* replaces mhc_layer_fwd_dynamic (bindings.cpp:880-952).  alpha_* point to
 * one device float each; b_res is [n,n].  token_state may be NULL for
 * inference (nothing saved).  1 <= n <= 32; which kernels run depends on n and
 * batch (n >= 8, or n = 6, 7 from 1024 tokens: the wide-rate set), so the
 * workspace size must come from the same (batch, n, hidden). */
MHC_API size_t mhc_layer_fwd_dynamic_workspace_bytes(int64_t batch, int32_t n, int64_t hidden);
MHC_API int mhc_layer_fwd_dynamic(const float* x, const float* rmsnorm_weight, const float* phi_pre,
                          const float* phi_post, const float* phi_res, const float* alpha_pre,
                          const float* alpha_post, const float* alpha_res, const float* b_pre,
                          const float* b_post, const float* b_res, float* out,
                          float* token_state, int64_t batch, int32_t n, int64_t hidden,
                          int32_t sinkhorn_iters, float sinkhorn_eps, float rmsnorm_eps,
                          void* workspace, size_t workspace_bytes, void* stream);

/* bf16 streams, an extension of mhc_layer_fwd_dynamic (the reference
 * keeps bf16 intermediates, bindings.cpp:906): x and out are bf16, the
 * parameters, token_state and all arithmetic fp32.  Needs n <= 4, hidden a
 * multiple of 64 and 16-byte aligned x / out / rmsnorm_weight
 * (MHC_ERR_UNSUPPORTED / MHC_ERR_ALIGNMENT otherwise).  Workspace as for
 * mhc_layer_fwd_dynamic. */
MHC_API int mhc_layer_fwd_dynamic_bf16(const void* x, const float* rmsnorm_weight,
                          const float* phi_pre, const float* phi_post, const float* phi_res,
                          const float* alpha_pre, const float* alpha_post,
                          const float* alpha_res, const float* b_pre, const float* b_post,
                          const float* b_res, void* out, float* token_state, int64_t batch,
                          int32_t n, int64_t hidden, int32_t sinkhorn_iters, float sinkhorn_eps,
                          float rmsnorm_eps, void* workspace, size_t workspace_bytes,
                          void* stream);

/* No counterpart in the reference.  Same as mhc_layer_fwd_dynamic, for
 * callers that cannot provide a workspace (no device allocator of their own,
 * device memory fixed at start-up, or a path that must not call cudaMalloc /
 * cudaFree because they can synchronise the device): the scratch comes from
 * a 16 MiB array in the library's device image, which every GPU that loads
 * the library holds until the process exits.  Requests needing more than
 * 16 MiB return MHC_ERR_UNSUPPORTED; the need depends on the shape, on
 * whether token_state is given (without it the record is scratch too) and on
 * the SM count -- on a 148-SM B200 at n=4, C=4096 about 20k tokens fit with a
 * token_state and about 16k without.  The first call on a
 * device looks up the array's device address (make it before any stream
 * capture).  All calls on a device share the array: calls whose kernels may
 * overlap on the GPU race and must be serialised by the caller. */
MHC_API int mhc_layer_fwd_dynamic_noalloc(const float* x, const float* rmsnorm_weight,
                                          const float* phi_pre, const float* phi_post,
                                          const float* phi_res, const float* alpha_pre,
                                          const float* alpha_post, const float* alpha_res,
                                          const float* b_pre, const float* b_post,
                                          const float* b_res, float* out, float* token_state,
                                          int64_t batch, int32_t n, int64_t hidden,
                                          int32_t sinkhorn_iters, float sinkhorn_eps,
                                          float rmsnorm_eps, void* stream);

/* replaces mhc_layer_bwd_dynamic (bindings.cpp:600-874).  All parameter
 * gradients are written (not accumulated); they are fixed-order reductions
 * over the batch, so results are bitwise reproducible run to run. */
MHC_API size_t mhc_layer_bwd_dynamic_workspace_bytes(int64_t batch, int32_t n, int64_t hidden);
MHC_API int mhc_layer_bwd_dynamic(const float* grad_out, const float* x, const float* rmsnorm_weight,
                          const float* phi_pre, const float* phi_post, const float* phi_res,
                          const float* alpha_pre, const float* alpha_post,
                          const float* alpha_res, const float* b_pre, const float* b_post,
                          const float* b_res, const float* token_state, float* grad_x,
                          float* grad_rmsnorm_weight, float* grad_phi_pre,
                          float* grad_phi_post, float* grad_phi_res, float* grad_alpha_pre,
                          float* grad_alpha_post, float* grad_alpha_res, float* grad_b_pre,
                          float* grad_b_post, float* grad_b_res, int64_t batch, int32_t n,
                          int64_t hidden, int32_t sinkhorn_iters, float sinkhorn_eps,
                          float rmsnorm_eps, void* workspace, size_t workspace_bytes,
                          void* stream);

/* bf16 streams for the backward: grad_out, x and grad_x are bf16, every
 * parameter gradient fp32 (arithmetic fp32, moments fp64 as in
 * mhc_layer_bwd_dynamic).  Needs n == 4, hidden a multiple of 32 and 16-byte
 * aligned tensors.  Workspace as for mhc_layer_bwd_dynamic. */
MHC_API int mhc_layer_bwd_dynamic_bf16(const void* grad_out, const void* x,
                          const float* rmsnorm_weight, const float* phi_pre,
                          const float* phi_post, const float* phi_res,
                          const float* alpha_pre, const float* alpha_post,
                          const float* alpha_res, const float* b_pre, const float* b_post,
                          const float* b_res, const float* token_state, void* grad_x,
                          float* grad_rmsnorm_weight, float* grad_phi_pre,
                          float* grad_phi_post, float* grad_phi_res, float* grad_alpha_pre,
                          float* grad_alpha_post, float* grad_alpha_res, float* grad_b_pre,
                          float* grad_b_post, float* grad_b_res, int64_t batch, int32_t n,
                          int64_t hidden, int32_t sinkhorn_iters, float sinkhorn_eps,
                          float rmsnorm_eps, void* workspace, size_t workspace_bytes,
                          void* stream);

/* ---------------------------------------------------------------------------
 * Fused mHC layer, static H (shared logits H_pre[n], H_post[n], H_res[n,n]).
 * The reference composes this from four operators (layer.py:142-170); these
 * entry points run the same math as one forward kernel and a fused backward.
 * The forward saves rms[batch] (RMSNorm denominators) when rms != NULL.
 * x/out are fp32 (..._f32) or bf16 with fp32 arithmetic (..._bf16).
 * ------------------------------------------------------------------------- */
MHC_API size_t mhc_layer_static_workspace_bytes(int64_t batch, int32_t n, int64_t hidden);
MHC_API int mhc_layer_fwd_static_f32(const float* x, const float* rmsnorm_weight, const float* H_pre,
                             const float* H_post, const float* H_res, float* out, float* rms,
                             int64_t batch, int32_t n, int64_t hidden, int32_t sinkhorn_iters,
                             float sinkhorn_eps, float rmsnorm_eps, void* workspace,
                             size_t workspace_bytes, void* stream);
MHC_API int mhc_layer_fwd_static_bf16(const void* x, const float* rmsnorm_weight, const float* H_pre,
                              const float* H_post, const float* H_res, void* out, float* rms,
                              int64_t batch, int32_t n, int64_t hidden, int32_t sinkhorn_iters,
                              float sinkhorn_eps, float rmsnorm_eps, void* workspace,
                              size_t workspace_bytes, void* stream);
MHC_API int mhc_layer_bwd_static(const float* grad_out, const float* x, const float* rmsnorm_weight,
                         const float* H_pre, const float* H_post, const float* H_res,
                         const float* rms, float* grad_x, float* grad_rmsnorm_weight,
                         float* grad_H_pre, float* grad_H_post, float* grad_H_res,
                         int64_t batch, int32_t n, int64_t hidden, int32_t sinkhorn_iters,
                         float sinkhorn_eps, float rmsnorm_eps, void* workspace,
                         size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Embedding lookup into residual streams, and its gradient.  No counterpart in
 * the reference, whose models start from embeddings made elsewhere.
 *   out[t, i, :] = scales[i] * weight[ids[t], :]        t < tokens, i < n <= 32
 * ids are int64 (ids_64 != 0) or int32; weight [vocab, hidden] and out
 * [tokens, n, hidden] are fp32 or bf16 each (products in fp32, rounded once);
 * scales is a HOST array of n floats, read before the call returns.  An id
 * outside [0, vocab) gives a row of NaN and reads nothing.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_stream_embedding_fwd(const void* ids, int32_t ids_64, const void* weight, int32_t weight_bf16,
                             void* out, int32_t out_bf16, const float* scales, int64_t tokens,
                             int32_t n, int64_t hidden, int64_t vocab, void* stream);
/* grad_weight[v, :] = sum over t with ids[t] = v, v != padding_idx, of
 * sum_i scales[i] grad_out[t, i, :], fp32 sums in a fixed order (bitwise
 * reproducible; token order within chunks, then the chunks' sums); the whole
 * [vocab, hidden] gradient is written, rows without a token as zeros.  Ids outside [0, vocab) add nothing; padding_idx < 0: none.
 * grad_weight must be 16-byte aligned. */
MHC_API size_t mhc_stream_embedding_bwd_workspace_bytes(int64_t tokens, int64_t hidden);
MHC_API int mhc_stream_embedding_bwd(const void* grad_out, int32_t g_bf16, const void* ids, int32_t ids_64,
                             void* grad_weight, int32_t gw_bf16, const float* scales, int64_t tokens,
                             int32_t n, int64_t hidden, int64_t vocab, int64_t padding_idx,
                             void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Activation checkpoints in 8 bits.  No counterpart in the reference, which
 * saves whole bf16 copies (ops.py:394-470).
 * A row of cols values is kept as int8 codes, padded with zeros to
 * mhc_checkpoint8_pitch(cols) = 128 * ceil(cols / 128) bytes, and one exponent
 * byte E per 32 codes (pitch / 32 a row): a code stands for code * 2^(E - 127).
 * With a = max |x| of a block, E >= 1 is the smallest with
 * a < 127.5 * 2^(E - 127), and code = x / 2^(E - 127) rounded to nearest, ties
 * to even (at E = 249 held to +-63: 64 would stand for 2^128).  E = 255: the
 * block held an infinity or a NaN and stands for NaNs.
 * codes must be 16-byte and exponents 4-byte aligned.
 * ------------------------------------------------------------------------- */
MHC_API int64_t mhc_checkpoint8_pitch(int64_t cols);
/* x [rows, cols] fp32 or bf16, rows row_stride elements apart */
MHC_API int mhc_checkpoint8_pack(const void* x, int32_t x_bf16, int64_t row_stride, int8_t* codes,
                         uint8_t* exponents, int64_t rows, int64_t cols, void* stream);
/* out [rows, cols] contiguous, fp32 or bf16 (both exact) */
MHC_API int mhc_checkpoint8_unpack(const int8_t* codes, const uint8_t* exponents, void* out,
                           int32_t out_bf16, int64_t rows, int64_t cols, void* stream);
/* RMSNorm (mhc_rmsnorm_fwd) of x [rows, cols] fp32 or bf16, out in x's type,
 * that also packs x in the same pass. */
MHC_API int mhc_rmsnorm_checkpoint8_fwd(const void* x, int32_t x_bf16, const float* weight, void* out,
                                float* rms, int8_t* codes, uint8_t* exponents, int64_t rows,
                                int64_t cols, float eps, void* stream);
/* Its backward at the restored input xh (rms is the forward's):
 *   grad_x = (g w - xh sum(g w xh) / (cols rms^2)) / rms, in g's type
 *   grad_weight = sum over rows of g xh / rms (fixed order) */
MHC_API size_t mhc_rmsnorm_checkpoint8_bwd_workspace_bytes(int64_t rows, int64_t cols);
MHC_API int mhc_rmsnorm_checkpoint8_bwd(const void* grad_out, int32_t g_bf16, const int8_t* codes,
                                const uint8_t* exponents, const float* weight, const float* rms,
                                void* grad_x, float* grad_weight, int64_t rows, int64_t cols,
                                void* workspace, size_t workspace_bytes, void* stream);
/* Weight gradient of a linear layer from its kept input:
 *   grad_weight[o, k] = sum_t grad_out[t, o] xh[t, k]        [out_features, in_features]
 * grad_out [tokens, out_features] fp32 or bf16, rows row_stride elements apart;
 * grad_weight fp32 or bf16, contiguous.  fp32 grad_out is used in full
 * precision; sums are fp32 and in a fixed order.  The workspace is smaller for a
 * bf16 grad_out whose start is 16-byte aligned and whose row_stride is a multiple
 * of 8 (g_aligned): any other is copied there first. */
MHC_API size_t mhc_checkpoint8_weight_grad_workspace_bytes(int64_t tokens, int64_t out_features,
                                                   int64_t in_features, int32_t g_bf16, int32_t g_aligned);
MHC_API int mhc_checkpoint8_weight_grad(const void* grad_out, int32_t g_bf16, int64_t row_stride,
                                const int8_t* codes, const uint8_t* exponents, void* grad_weight,
                                int32_t gw_bf16, int64_t tokens, int64_t out_features,
                                int64_t in_features, void* workspace, size_t workspace_bytes,
                                void* stream);

/* ---------------------------------------------------------------------------
 * Dropout from a counter-based generator.  No counterpart in the reference, whose
 * layers draw no random numbers.
 *   out[i] = number(i) < drop ? 0 : x[i] / (1 - drop / 65536)       i < count
 * x and out fp32 or bf16 (products in fp32, rounded once); 0 <= drop <= 65536, the
 * probability in 65536ths.  number(i) is 16-bit number i % 8 of group
 * position + i / 8 (mod 2^64) of the seed's stream: Philox4x32-10 at counter
 * (group low, group high, 0, 0), key (seed low, seed high), word by word, low half
 * first.  state, if not NULL, points to two device words (seed, position), read by
 * the kernel in place of the arguments.  The backward pass is the same call on the
 * gradient; nothing is stored.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_dropout(const void* x, int32_t x_bf16, void* out, int64_t count, int32_t drop,
                        const uint64_t* state, uint64_t seed, uint64_t position, void* stream);
/* out[0..1] = state[0..1], then state[1] += groups (one atomic step, so that a
 * captured graph takes new numbers each time, and overlapping calls different ones) */
MHC_API int mhc_dropout_take(uint64_t* state, uint64_t* out, int64_t groups, void* stream);

/* ---------------------------------------------------------------------------
 * Residual addition and RMSNorm.  The reference normalises by itself
 * (ops.py:87-136).  Rows of cols values, contiguous:
 *   hidden = residual + dropout(branch)          (mhc_dropout's numbers, i = row cols + col)
 *   r = sqrt(mean hidden^2 + eps),  out = hidden / r * weight
 * residual and hidden have one type, branch and out another (fp32 or bf16 each);
 * the norm is of hidden as it is returned.  rms [rows] may be NULL.  codes and
 * exponents, if not NULL, receive out in 8 bits as mhc_checkpoint8_pack(out) does.
 * hidden and out may not overlap the inputs.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_add_rmsnorm_fwd(const void* residual, int32_t residual_bf16, const void* branch,
                                int32_t branch_bf16, const float* weight, void* hidden, void* out,
                                float* rms, int8_t* codes, uint8_t* exponents, int64_t rows,
                                int64_t cols, float eps, int32_t drop, const uint64_t* state,
                                uint64_t seed, uint64_t position, void* stream);
/* The same without dropout, the output as 8-bit codes [rows, cols] (e4m3, or int8 if
 * codes_int8) with fp32 scales: one a row, or, if grouped, one for each 128 columns
 * [rows, ceil(cols / 128)].  With a = max |out| of a group, scale =
 * max(a / 448, 2^-100) (int8: a / 127) and code = out / scale rounded to nearest,
 * ties to even; a group with an infinity or a NaN, also of hidden * weight, which is
 * formed in fp32, has a NaN scale. */
MHC_API int mhc_add_rmsnorm_coded(const void* residual, int32_t residual_bf16, const void* branch,
                                  int32_t branch_bf16, const float* weight, void* hidden,
                                  void* codes, int32_t codes_int8, float* scales, int32_t grouped,
                                  int64_t rows, int64_t cols, float eps, void* stream);
/* out = code * scale [rows, cols] */
MHC_API int mhc_coded8_unpack(const void* codes, int32_t codes_int8, const float* scales,
                              int32_t grouped, void* out, int32_t out_bf16, int64_t rows,
                              int64_t cols, void* stream);
/* Backward of mhc_add_rmsnorm_fwd from its hidden and rms:
 *   gi = grad_hidden + (g w - hidden sum(g w hidden) / (cols r^2)) / r,  g = grad_out
 *   grad_residual = gi,  grad_branch = dropout(gi),  grad_weight = sum over rows of g hidden / r
 * grad_hidden may be NULL (zero), grad_branch too (not wanted: without dropout and
 * with one type it equals grad_residual).  grad_weight's sums have a fixed order. */
MHC_API size_t mhc_add_rmsnorm_bwd_workspace_bytes(int64_t rows, int64_t cols);
MHC_API int mhc_add_rmsnorm_bwd(const void* grad_hidden, const void* grad_out, const void* hidden,
                                int32_t residual_bf16, int32_t branch_bf16, const float* weight,
                                const float* rms, void* grad_residual, void* grad_branch,
                                float* grad_weight, int64_t rows, int64_t cols, int32_t drop,
                                const uint64_t* state, uint64_t seed, uint64_t position,
                                void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Log probabilities of given tokens, entropy and alternatives.  No counterpart in
 * the reference.  logits [rows, vocab] fp32 or bf16, rows row_stride elements apart,
 * vocab <= 2^21; targets int64 (targets_64 != 0) or int32.  With m = max x and
 * s = sum exp(x - m) of a row:
 *   logprob = x[target] - m - ln s,   entropy = -sum p ln p  (0 ln 0 = 0)
 *   top_id, top_logprob [rows, top]: the `top` <= 32 largest logits, largest first,
 *   ties (and +0, -0) to the lowest index; NaNs come last
 *   stats [rows, 2] = (m, s), what the backward needs beside the entropy
 * A target equal to ignore_index has logprob 0, any other outside [0, vocab) NaN.  A
 * logit of -inf has probability 0; a row of nothing else has logprobs -inf and
 * entropy 0.  A row with +inf or NaN has logprob, entropy and top_logprob NaN.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_token_logprobs_fwd(const void* logits, int32_t logits_bf16, int64_t row_stride,
                                   const void* targets, int32_t targets_64, int64_t ignore_index,
                                   float* logprob, float* entropy, float* top_logprob,
                                   int64_t* top_id, float* stats, int64_t rows, int64_t vocab,
                                   int32_t top, void* stream);
/* Gradient of the logits [rows, vocab], contiguous, in their type, from the
 * gradients of the three results (each may be NULL; grad_top and top_id [rows, top]
 * with top > 0).  A row of nothing but -inf gets zeros; a target outside
 * [0, vocab) other than ignore_index gives its row NaNs if grad_logprob is given
 * (the other results do not depend on it). */
MHC_API int mhc_token_logprobs_bwd(const void* logits, int32_t logits_bf16, int64_t row_stride,
                                   const void* targets, int32_t targets_64, int64_t ignore_index,
                                   const float* stats, const float* entropy, const int64_t* top_id,
                                   const float* grad_logprob, const float* grad_entropy,
                                   const float* grad_top, void* grad_logits, int64_t rows,
                                   int64_t vocab, int32_t top, void* stream);

/* ---------------------------------------------------------------------------
 * Device error word.  No counterpart in the reference.  Kernels that wait on
 * asynchronous copies (TMA + mbarrier) bound every wait; a wait that runs out
 * sets this word to nonzero and the kernel abandons its work (its outputs are
 * then incomplete) instead of hanging the GPU.  Reads the word (synchronous
 * copy from the device) and optionally resets it to zero.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_device_error_word(int32_t* value, int32_t reset);

/* ---------------------------------------------------------------------------
 * Kernel timing (tracing).  No counterpart in the reference, which times
 * whole calls from Python (benchmark.py:156-269).  While enabled, every kernel
 * this library launches is bracketed by two CUDA events on its own stream;
 * mhc_profile_report() waits for them and writes one line per kernel name:
 * "<name> <launches> <total_ms>\n" (NUL-terminated, truncated to cap), then
 * clears the record.  Returns the number of bytes written, or < 0 on error.
 * Process-wide; meant for benchmarking, not for concurrent production use.
 * ------------------------------------------------------------------------- */
MHC_API int mhc_profile_enable(int enable);
MHC_API int mhc_profile_report(char* buf, size_t cap);

#ifdef __cplusplus
}
#endif

#endif /* MHC_B200_H_ */

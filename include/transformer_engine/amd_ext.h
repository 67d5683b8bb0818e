/* Extensions with NO counterpart in the reference.  They exist because this
 * library is also bound from languages that cannot catch C++ exceptions or build
 * std::vector arguments (ctypes, cgo, JNI ...).
 */
#ifndef TE_AMD_EXT_H_
#define TE_AMD_EXT_H_

#include "transformer_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Error mode.  0 (default) = reference behaviour: a failed check throws
 * std::runtime_error through the C entry point (ref common/util/logging.h:38-51).
 * 1 = "record": the entry point catches the exception, stores its text in a
 * thread-local slot and returns normally; the caller polls nvte_amd_last_error(). */
void nvte_amd_set_error_mode(int mode);
int nvte_amd_get_error_mode(void);
/* Text of the last recorded error on this thread, or NULL.  Valid until the next
 * nvte_* call on the same thread. */
const char *nvte_amd_last_error(void);
void nvte_amd_clear_error(void);
/* Address of a process-wide count of recorded errors (all threads).  A foreign-function binding reads it
 * before and after a call - a plain memory read - and only asks for nvte_amd_last_error() when it moved:
 * polling the thread-local slot through a second foreign call after EVERY call doubled the per-call cost of
 * the ctypes binding. */
const unsigned long long *nvte_amd_error_counter(void);

/* Plain-C twin of nvte_delayed_scaling_recipe_amax_and_scale_update_after_reduction
 * (ref recipe.h:71-74, whose std::vector arguments make the symbol C++-mangled). */
void nvte_amd_delayed_scaling_after_reduction(const NVTETensor amax_reduction_buffer,
                                              const NVTETensor *amax_histories,
                                              const NVTETensor *scales, size_t num_tensors,
                                              const char *amax_compute_algo,
                                              enum NVTEDType fp8_dtype, float margin,
                                              hipStream_t stream);

/* The same bulk update with ONE FP8 format per tensor, so that the forward (E4M3) and backward (E5M2 under
 * the HYBRID format) recipe states of a step share one launch: the reference issues one call per direction
 * (ref pytorch/quantization.py:646-701, recipe.h:71-74); a layer's two states are independent, so updating
 * both behind the backward pass gives the values of the two separate calls. */
void nvte_amd_delayed_scaling_after_reduction_multi(const NVTETensor amax_reduction_buffer,
                                                    const NVTETensor *amax_histories,
                                                    const NVTETensor *scales,
                                                    const enum NVTEDType *fp8_dtypes,
                                                    size_t num_tensors, const char *amax_compute_algo,
                                                    float margin, hipStream_t stream);

/* MXFP8 "transposed columnwise" layout (no counterpart in the reference; OPTIONAL since round 3).
 * The reference keeps the columnwise-quantized MXFP8 payload in the input's own [rows, cols]
 * layout and lets cuBLASLt read it as a non-TN operand; nvte_cublas_gemm* here read that layout
 * K-major through the transposing LDS loads (the default, nothing to set).  An MXFP8 output tensor
 * can instead ask nvte_quantize* to store its columnwise payload transposed (K-contiguous):
 *   columnwise_data       [cols, rows]              (FP8 bytes, blocks of 32 along the LAST dim)
 *   columnwise_scale_inv  [pad128(cols), pad4(ceil(rows/32))]   (e8m0; GEMM-swizzled if the
 *                          tensor's with_gemm_swizzled_scales flag is set -- for that flag the
 *                          bytes are identical to the reference's swizzled columnwise scales)
 * nvte_cublas_gemm* consume either layout for the NN / NT layouts (dgrad / wgrad).  Default 0 =
 * reference layout. */
void nvte_amd_set_columnwise_transposed(NVTETensor tensor, int transposed);
int nvte_amd_get_columnwise_transposed(const NVTETensor tensor);

/* The same for a grouped MXFP8 tensor (no counterpart in the reference): columnwise_data holds every
 * member's payload transposed ([last, first_i] at the member's element offset) and
 * columnwise_scale_inv the members' [pad128(last), pad4(first_i / 32)] scale matrices back to back
 * (member i at the sum of the padded sizes before it - the offset rule of ref
 * gemm/cublaslt_grouped_gemm.cu:1117-1198).  nvte_group_quantize writes this layout when the flag is set;
 * nvte_grouped_gemm* takes it or the reference's un-transposed columnwise members (read K-major, members
 * with one last dimension) for the NN / NT layouts (dgrad / wgrad).  Member first dims must be
 * multiples of 128 for grouped MXFP8 tensors (the reference states the same for the logical first dim,
 * cast/mxfp8/group_quantize_mxfp8.cuh:842, and its swizzled-scale offsets assume it per member). */
void nvte_amd_set_grouped_columnwise_transposed(NVTEGroupedTensor tensor, int transposed);
int nvte_amd_get_grouped_columnwise_transposed(const NVTEGroupedTensor tensor);

/* A list of independent GEMMs in ONE persistent launch (no counterpart in the reference, whose list form
 * nvte_multi_tensor_gemm, gemm/cublaslt_gemm.cu:1052, spreads the list over streams and shares one
 * transa / transb): entry i computes D[i] = op(A[i]) op(B[i]) (+ D[i] when accumulate[i]) exactly as
 * nvte_cublas_gemm(A[i], B[i], D[i], NULL, NULL, transa[i], transb[i], grad, workspace, accumulate[i], ...)
 * does.  Meant for the dgrad + wgrad pair of a layer: the tiles of all entries form one list that the
 * persistent workgroups walk, cut per XCD by cost, so a GEMM whose tile count is not a multiple of the
 * workgroup count (wgrad of Llama-3-8B's FFN: 3.5 rounds) leaves no idle half round.  Taken when 2 <= num_gemms
 * <= 8, every operand is FP8 with per-tensor scaling, the FP8 formats and the (high-precision) output dtype
 * agree across the list and workspace holds nvte_get_grouped_gemm_setup_workspace_size(num_gemms) bytes;
 * any other list runs as the nvte_cublas_gemm calls above, one after the other.  accumulate may be NULL. */
void nvte_amd_multi_gemm(const NVTETensor *A, const NVTETensor *B, NVTETensor *D, const int *transa,
                         const int *transb, int num_gemms, int grad, NVTETensor workspace, const int *accumulate,
                         hipStream_t stream);

/* ---- Global gradient norm and clipping over a list of tensors (Python: weight_update.grad_norm, clip_grad_norm).
 * norm = sqrt(sum of squares of every element of every tensor), squares summed in 64 bits in a fixed order.
 * grads[i] is a device array of numels[i] elements of NVTEDType dtypes[i] (fp32 / fp16 / bf16, mixed at will); empty
 * tensors count nothing.  The lists themselves are host arrays.  Inf and NaN run through: the norm is then Inf or NaN. */
size_t nvte_amd_grad_norm_workspace_size(const size_t *numels, size_t num_tensors);
/* *sum_of_squares (fp64) and *norm (fp32), device pointers; either may be NULL */
void nvte_amd_grad_norm(const void *const *grads, const size_t *numels, const int *dtypes, size_t num_tensors,
                        double *sum_of_squares, float *norm, void *workspace, size_t workspace_bytes, hipStream_t stream);
/* outs[i] = grads[i] * min(1, max_norm / (norm + eps)), rounded once to out_dtypes[i]; *norm as above.  outs[i] may be
 * grads[i] itself (in place, one dtype); any other overlap of an output with a tensor of the call is an error. */
void nvte_amd_clip_grad_norm(const void *const *grads, void *const *outs, const size_t *numels, const int *dtypes,
                             const int *out_dtypes, size_t num_tensors, float max_norm, float eps, float *norm,
                             void *workspace, size_t workspace_bytes, hipStream_t stream);
/* The second half alone, for a sum of squares that was added up over ranks first. */
void nvte_amd_clip_by_sum_of_squares(const void *const *grads, void *const *outs, const size_t *numels, const int *dtypes,
                                     const int *out_dtypes, size_t num_tensors, const double *sum_of_squares,
                                     float max_norm, float eps, float *norm, hipStream_t stream);

/* ---- Low-rank adapters of many requests beside a shared projection (Python: lora.py).
 * x [tokens, in], a [num_adapters, rank, in], b [num_adapters, out, rank], base / out [tokens, out], all of one dtype (bf16 or
 * fp16), contiguous; up to 2^27 tokens; adapter_ids [tokens] int32, any order, a value outside [0, num_adapters) = no adapter; scaling
 * [num_adapters] fp32 or NULL (1); base NULL = zero, or out itself.  rank 1 to 128, any feature sizes.
 *   low[t] = a[id] x[t]        out[t] = base[t] + scaling[id] b[id] low[t]
 * low [nvte_amd_lora_num_slices(tokens, in), tokens, rank] fp32: partial sums of the rank vectors, which the backward pass reads
 * (rows without an adapter are not written).  A non-finite weight or activation makes its own rows non-finite and no other; where
 * the sum would be Inf it may be NaN. */
size_t nvte_amd_lora_num_slices(size_t tokens, size_t features);
size_t nvte_amd_lora_forward_workspace_size(size_t tokens, size_t num_adapters);   /* 0: workspace may be NULL */
void nvte_amd_lora_forward(const void *x, const void *a, const void *b, const int *adapter_ids, const float *scaling,
                           const void *base, void *out, float *low, size_t tokens, size_t in_features, size_t out_features,
                           size_t rank, size_t num_adapters, int dtype, void *workspace, size_t workspace_bytes,
                           hipStream_t stream);
/* dx[t] = base_grad[t] + scaling[id] a[id]^T (b[id]^T dy[t]); da [num_adapters, rank, in] and db [num_adapters, out, rank], in
 * dtype or fp32 (grad_dtype), are sums over each adapter's tokens in a fixed order, zero for an adapter without tokens.  dx may
 * be NULL, da and db may be NULL together; base_grad NULL = zero, or dx itself.  Up to 4096 adapters when da / db are wanted.
 * The first size is that of a call with da and db, the second (a part of it) that of a call without them. */
size_t nvte_amd_lora_backward_workspace_size(size_t tokens, size_t in_features, size_t out_features, size_t rank,
                                             size_t num_adapters);
size_t nvte_amd_lora_dgrad_workspace_size(size_t tokens, size_t out_features, size_t rank, size_t num_adapters);
void nvte_amd_lora_backward(const void *x, const void *dy, const void *a, const void *b, const int *adapter_ids,
                            const float *scaling, const float *low, const void *base_grad, void *dx, void *da, void *db,
                            size_t tokens, size_t in_features, size_t out_features, size_t rank, size_t num_adapters,
                            int dtype, int grad_dtype, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* ---- A mixture-of-experts layer for a few tokens (Python: moe.py); larger batches: the grouped GEMM.
 * Router (up to 2^26 - 4 tokens): p = softmax(logits[t]) over num_experts (<= 1024) fp32 / fp16 / bf16 logits; topk_ids [tokens, top_k] int32 = the largest,
 * in falling order, ties to the lowest index, NaN last; topk_weights fp32 = p of them, divided by their sum if renormalize. */
void nvte_amd_moe_topk(const void *logits, int *topk_ids, float *topk_weights, size_t tokens, size_t num_experts, size_t top_k,
                       int renormalize, int dtype, hipStream_t stream);
/* out[t] = sum_j topk_weights[t, j] w_fc2[e] (silu(w_fc1[e][:ffn] x[t]) * (w_fc1[e][ffn:] x[t])), e = topk_ids[t, j]; an id
 * outside [0, num_experts) adds nothing.  x, out [tokens, hidden] bf16 or fp16; w_fc1 [num_experts, 2 ffn, hidden] and w_fc2
 * [num_experts, hidden, ffn] of the same dtype, or FP8 E4M3 with one fp32 scale_inv per expert.  Up to 256 tokens, top_k up to
 * 64, tokens * top_k up to 4096.  out must not overlap an input.  Non-finite values as above: those of one token or expert stay
 * with the tokens that meet them. */
size_t nvte_amd_moe_forward_workspace_size(size_t tokens, size_t top_k, size_t num_experts, size_t hidden, size_t ffn);
void nvte_amd_moe_forward(const void *x, const void *w_fc1, const void *w_fc2, const float *fc1_scale_inv,
                          const float *fc2_scale_inv, const int *topk_ids, const float *topk_weights, void *out,
                          size_t tokens, size_t top_k, size_t num_experts, size_t hidden, size_t ffn, int dtype,
                          int weight_dtype, void *workspace, size_t workspace_size, hipStream_t stream);

/* Library identification: "transformerengine_amd <version> gfx950". */
const char *nvte_amd_version(void);

#ifdef __cplusplus
}
#endif
#endif

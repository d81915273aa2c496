// C++ interface behind the C ABI's forward entries: what the ABI unit offers to the package's own host layers (the
// Python binding), which know more about a call than the C entries can say -- the element types of activations and
// outputs, and that the weights were in place before the stream's previous kernel started (launch overlap).
#pragma once

#include <stdint.h>

#include "../../include/lloom_b200.h"

namespace lloom {

// The setting of lloom_b200_set_launch_overlap: 1 on, 0 off, -1 neither (the host layer decides call by call).
int launch_overlap();

struct FwdIo {
    int x_type = LLOOM_F32, y_type = LLOOM_F32;  // LLOOM_F32 / LLOOM_F16 / LLOOM_BF16
    // The call's kernels may start before their stream predecessor has finished; they read nothing but weights until it
    // has.  Only for weights that no work still in flight writes.
    bool overlap = false;
};

// All return a status code; shapes, pointers and workspace are checked as by the C entries of the same name.
// lloom_b200_qmatmul_fwd (w_image == nullptr, store == LLOOM_STORE_PLAIN), _image and _store in one.
int qmatmul_forward(int w_dtype, const void *w_blocks, const void *w_image, const void *x, void *y, int64_t m, int64_t n, int64_t k,
                    int64_t ldy, int store, void *workspace, int64_t workspace_bytes, void *stream, const FwdIo &io);
// The same from canonical activation blocks (lloom_b200_qmatmul_fwd_acts); io.x_type does not count
int qmatmul_forward_acts(int w_dtype, const void *w_blocks, const void *w_image, const void *act, void *y, int64_t m, int64_t n, int64_t k,
                         int64_t ldy, void *workspace, int64_t workspace_bytes, void *stream, const FwdIo &io);
// Exactly one of act (canonical activation blocks) and x is non-null
int qmatmul_forward_group(int w_dtype, int n_mats, const void *const *w_blocks, const void *act, const void *x, float *const *ys,
                          const int64_t *ns, const int64_t *ldys, const int *stores, int64_t m, int64_t k, void *workspace, int64_t workspace_bytes,
                          void *stream, const FwdIo &io);
// ids: 32-bit, or 64-bit of which the low half counts
int indexed_moe_forward(int w_dtype, const void *w_experts, int64_t n_experts, int64_t n, int64_t k, const float *x, int64_t batch,
                        int64_t in_dim1, const void *ids, bool ids64, int64_t topk, float *out, void *workspace,
                        int64_t workspace_bytes, void *stream, const FwdIo &io);
int get_rows(int dtype, const void *blocks, int64_t rows, int64_t hidden, const void *ids, bool ids64, int64_t n_ids, float *out,
             void *stream, bool overlap);
// lloom_b200_rms_norm, lloom_b200_dequantize_act (norm.cu)
int rms_norm(const void *x, const void *residual, const void *weight, int x_type, int w_type, double eps, int64_t m, int64_t k, int64_t ldx,
             int64_t ldr, void *h, void *y, int y_type, void *stream, bool overlap);
int dequantize_act(int act_dtype, const void *act_blocks, int64_t elem_count, float *out, void *stream, bool overlap);
// The microscaled 4-bit entries of the same names (mx.cu); overlap in mx_forward: the weights are in place
int mx_quantize(const void *x, int x_type, int64_t rows, int64_t k, void *image, int64_t image_bytes, void *stream, bool overlap);
int mx_dequantize(const void *image, int64_t rows, int64_t k, void *out, bool f16, void *stream, bool overlap);
int mx_forward(const void *image, const void *x, int x_type, void *y, int y_type, int64_t m, int64_t n, int64_t k, int64_t ldy, void *workspace,
               int64_t workspace_bytes, void *stream, bool overlap);

// lloom_b200_sample (sample.cu)
int sample(const void *logits, int type, int64_t batch, int64_t vocab, int64_t ld, const float *u, const float *temperature, double temperature_all,
           const int *top_k, int64_t top_k_all, const float *top_p, double top_p_all, const float *min_p, double min_p_all, int64_t *ids,
           float *probs, void *stream, bool overlap);

}  // namespace lloom

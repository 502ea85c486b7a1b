// internal.h — declarations shared by the library's translation units (not part of the C ABI).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>
#include <string>

#include "snb_matmul.h"

namespace snb {

// One product with its epilogue, after argument validation; element types are SNB_TYPE_*.
struct GemmRequest {
    snb_product p;
    uint64_t count;
    int a_type, b_type, c_type;
    int precision;
    const void* A;
    const void* B;
    void* C;
    const float* bias;
    int activation;
    int aux_type;
    void* pre;
    const void* gelu_input;
    const void* residual;
    int causal;
    int64_t causal_offset;
    const float* row_scale;   // [rows] output-row multipliers (count 1), or nullptr
    bool deterministic;       // split-K partials summed in a fixed order (SNB_GEMM_DETERMINISTIC)
    const snb_head_layout* a_heads;  // left operand read from its head-major form, or nullptr (snb_gemm_args)
    const snb_head_layout* c_heads;  // output written head-major, or nullptr
    int sm_budget;            // SMs the persistent grid may occupy (0: all; snb_set_sm_budget)
    uint64_t c_ld;            // elements between the output's rows (0: cols); other than cols on the tensor cores only,
                              // for one plain product (no split of K, no tensor laid out like the output)
    // f32 operands split in two planes (TF32 precision, count 1, f32 output, not deterministic): A and B point to the
    // first plane, the second lies plane_stride elements after it, and `low` says which one holds the low parts.
    // split_inner: longest sum of products of leading parts (see gemm_tc.cuh). 0: ordinary operands.
    uint64_t split_inner, a_plane_stride, b_plane_stride;
    int a_low, b_low;
};

struct DeviceInfo {
    int device;
    int sm_count;
    int major, minor;
};

// Properties of the current device (cached per device).
int current_device_info(DeviceInfo* info, std::string* err);

// Runs the product on a tcgen05 kernel if its layout allows TMA (unit strides, 16-byte alignment); *launched
// says whether it did and *path which kernel (SNB_PATH_TENSOR_CORE or SNB_PATH_TENSOR_CORE_PAIR). Returns SNB_OK
// or an error code (with *err set).
int tc_gemm_try(cudaStream_t stream, const GemmRequest& r, bool* launched, int* path, std::string* err);

// Runs the product on the strided SIMT kernel (any layout).
int simt_gemm(cudaStream_t stream, const GemmRequest& r, std::string* err);

int causal_softmax(cudaStream_t stream, float* scores, uint64_t rows, uint64_t queries, uint64_t keys, float scale,
                   uint64_t query_offset, uint16_t* probs_bf16, std::string* err);
int softmax_backward(cudaStream_t stream, const float* probabilities, float* grad, uint64_t rows, uint64_t cols,
                     std::string* err);
int causal_softmax_backward(cudaStream_t stream, const float* probabilities, float* grad, uint64_t rows,
                            uint64_t queries, uint64_t cols, uint64_t query_offset, uint16_t* grad_bf16,
                            std::string* err);

// Fused causal attention forward (tcgen05; head_dim 64; bf16 q/k/v [count, rows, 64]).
int fused_attention_forward(cudaStream_t stream, const void* q, const void* k, const void* v, uint64_t count,
                            uint64_t queries, uint64_t keys, float scale, uint64_t query_offset, void* out,
                            int out_type, float* lse, std::string* err);
// Softmax cross-entropy with its gradient over `heads` classifiers side by side (cross_entropy.cu): head h owns
// columns column_offset + h * classes .. and target target_offset + h of each target row. row_losses
// ([rows * heads], head fastest) and loss_sums ([heads], added to) may be null; grad may alias logits when the
// element types match.
int cross_entropy_launch(cudaStream_t stream, const void* logits, int logits_type, uint64_t rows, uint64_t row_width,
                         const uint32_t* targets, uint64_t target_stride, uint64_t heads, uint64_t column_offset,
                         uint64_t classes, uint64_t target_offset, const float* grad_scales, float grad_scale,
                         float* row_losses, float* loss_sums, void* grad, int grad_type, std::string* err);

// RMSNorm and optimizer launches (norm_optim.cu).
int rms_norm_forward_launch(cudaStream_t s, const void* input, int input_type, const float* gain, void* output,
                            int output_type, float* inv_rms, uint64_t rows, uint64_t cols, float epsilon,
                            std::string* err);
int rms_norm_backward_launch(cudaStream_t s, const float* dy, const float* x, const float* gain, const float* inv_rms,
                             float* dx, float* gain_grad, uint64_t rows, uint64_t cols, std::string* err);
int scale_rows_launch(cudaStream_t s, const float* scale, const void* in, int in_type, void* out, int out_type,
                      uint64_t rows, uint64_t cols, std::string* err);
int adamw_launch(cudaStream_t s, float* parameter, const float* gradient, float* first, float* second, uint64_t count,
                 const snb_adamw_hyper& h, std::string* err);
int sum_of_squares_launch(cudaStream_t s, const float* values, uint64_t count, double* total, std::string* err);
int adamw_multi_launch(cudaStream_t s, const snb_adamw_tensor* tensors, uint64_t n, const snb_adamw_hyper& h,
                       float max_gradient_norm, double* square_sum, std::string* err);

// Fused causal attention backward (attention_fused_bwd.cuh): dq [count, queries, 64], dk and dv [count, keys, 64],
// all f32 and overwritten, from bf16 q, k, v, d_out, the forward's output (f32 or bf16) and its log-sum-exp. The
// row-statistics scratch comes from cudaMallocAsync on `stream`, or with static_scratch_only from a fixed
// __device__ array (no allocation; SNB_ERR_INVALID_ARGUMENT when it is too small; concurrent calls share it).
int fused_attention_backward(cudaStream_t stream, const void* q, const void* k, const void* v, const void* out,
                             int out_type, const void* d_out, const float* lse, uint64_t count, uint64_t queries,
                             uint64_t keys, float scale, uint64_t query_offset, float* dq, float* dk, float* dv,
                             bool static_scratch_only, std::string* err);

// The attention head permutes (heads.cu): split = packed -> head-major, else head-major -> packed; element types
// SNB_TYPE_*; the layout is checked by the caller.
int permute_heads_launch(cudaStream_t stream, bool split, const void* src, int src_type, void* dst, int dst_type,
                         const snb_head_layout& layout, std::string* err);

// Launches a one-thread kernel whose mbarrier wait nothing completes; it gives up after limit_ns.
int bounded_wait_probe(cudaStream_t stream, uint64_t limit_ns, std::string* err);

// Reads and clears the tensor-core kernels' device status word on the current device (synchronizes first).
int read_and_clear_device_status(unsigned int* status, std::string* err);

// One product of the vocabulary's softmax cross entropy (tc_gemm.cu): logits = A B for `classes` classes from
// class_begin on, A [rows, inner] (K-major, rows a_ld elements apart), B [classes, inner] (rows b_ld apart) or with
// b_mn_major [inner, classes]; bf16, or f32 on TF32 tensor cores. Without `grad` the row statistics are written
// (partials, target_logit); with it softmax minus one-hot, as bf16 [rows, grad_ld], or for f32 operands as the two
// f32 tensors grad and grad_low whose sum it is. Bases and row pitches are multiples of 16 bytes.
struct VocabProduct {
    int type;
    uint64_t rows, classes, inner;
    const void* A;
    uint64_t a_ld;
    const void* B;
    uint64_t b_ld;
    bool b_mn_major;
    const uint32_t* targets;
    int64_t class_begin;
    float2* partials;
    float* target_logit;
    // With the statistics: the targets' logits as rounded f32 sums of the operands as the caller has them; or null.
    float* exact_logit;
    const void* hidden;
    const void* weight;
    uint64_t hidden_row, weight_class, weight_inner, width;  // element strides
    uint64_t vocabulary;     // classes of the whole
    const float2* row_stats;
    void* grad;
    void* grad_low;
    uint64_t grad_ld;
    int sm_budget;
};
int tc_vocab_product(cudaStream_t stream, const VocabProduct& v, std::string* err);

// Softmax cross entropy over a vocabulary in pieces (vocab_loss.cu).
bool vocab_loss_few_rows(const snb_vocabulary_loss_args& a);  // whether the CUDA cores compute the logits
int vocab_loss_workspace(const snb_vocabulary_loss_args& a, uint64_t* bytes, std::string* err);
int vocab_loss_launch(cudaStream_t stream, const snb_vocabulary_loss_args& a, bool deterministic, int sm_budget,
                      std::string* err);

// Layer norm (layer_norm.cu).
int layer_norm_workspace(uint64_t rows, uint64_t cols, uint64_t* bytes, std::string* err);
int layer_norm_forward_launch(cudaStream_t stream, const snb_layer_norm_args& a, std::string* err);
int layer_norm_backward_launch(cudaStream_t stream, const snb_layer_norm_args& a, std::string* err);

// AdamW with 8-bit moments (adamw8.cu).
uint64_t adamw8_workspace(uint64_t tensor_count);
int adamw8_step_launch(cudaStream_t stream, const snb_adamw8_tensor* tensors, uint64_t n, const snb_adamw_hyper& h,
                       float max_gradient_norm, uint64_t seed, double* square_sum, double* partials, std::string* err);
int adamw8_moments_launch(cudaStream_t stream, const snb_adamw8_moments_out* tensors, uint64_t n, std::string* err);

std::string cuda_message(const char* what, cudaError_t e);

// The reference's seeded stream on the device (random.cu): normal values (f32 or bf16 output) and below(bound)
// integers from draw first_draw + 1 on.
int random_normal_launch(cudaStream_t s, void* out, int out_type, uint64_t count, uint64_t seed, uint64_t first_draw,
                         float stddev, std::string* err);
int random_below_launch(cudaStream_t s, uint32_t* out, uint64_t count, uint64_t seed, uint64_t first_draw,
                        uint64_t bound, std::string* err);

}  // namespace snb

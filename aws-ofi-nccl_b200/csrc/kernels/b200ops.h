// Entry points of libb200ops.so that the native layers (torch_ops.cpp) call. The sources that define them
// include this header too, so that a changed signature does not compile on one side only.
#pragma once

extern "C" {

int b200_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc,
                   int a_mn, int b_mn, int out_fp32, int accumulate, int bn, int max_ctas, void* stream);

// Both gradients of a linear layer; see gemm_grads.cu. *launches: kernels launched, 1 or 2.
int b200_linear_grads(const void* dy, const void* x, const void* w, void* dx, void* dw, int M, int N, int K, long long lddy,
                      long long ldx, long long ldw, long long lddx, long long lddw, int accumulate, int* launches, void* stream);

int b200_rmsnorm_fwd(const void* x, const void* res, void* h_out, const void* w, void* y, float* rstd, int T, int H, float eps,
                     void* stream);
int b200_embedding_fwd(const long long* ids, const void* table, void* out, long long T, int H, void* stream);
int b200_embedding_bwd(const long long* ids, const void* dout, void* dtable, long long T, int H, void* stream);
int b200_cross_entropy(void* logits, const long long* targets, float* loss, int T, int V, long long ld, float grad_scale, void* stream);
int b200_rmsnorm_bwd_partial_rows();
int b200_rmsnorm_bwd(const void* dy, const void* x, const void* w, const float* rstd, const void* dres, void* dx,
                     float* dw_partial, void* dw, int accumulate_dw, int T, int H, void* stream);

int b200_swiglu_fwd(const void* gu, void* out, long long T, int F, void* stream);
int b200_swiglu_bwd(const void* dout, const void* gu, void* dgu, long long T, int F, void* stream);

// gate|up = x w^T with act = silu(gate) * up, and the gradient at gate|up from dy and the down projection w; see
// gemm_swiglu.cu. The bwd call wants `scratch` [M][F] bf16 where b200_gemm_swiglu_bwd_launches says 2.
int b200_gemm_swiglu(const void* x, const void* w, void* gu, void* act, int M, int F, int K, long long ldx, void* stream);
int b200_gemm_swiglu_bwd(const void* dy, const void* w, const void* gu, void* dgu, void* scratch, int M, int F, int K, long long lddy,
                         void* stream);
int b200_gemm_swiglu_launches(const void* x, const void* w, int M, int F, int K, long long ldx);
int b200_gemm_swiglu_bwd_launches(const void* dy, const void* w, int M, int F, int K, long long lddy);

int b200_rope_qkv(void* qkv, long long pitch, void* q, void* k, void* v, const long long* strides, const float* cs,
                  const float* sn, long long T, int nq, int nkv, int hd, int seq, int backward, void* stream);

// RMSNorm with its output in 8 bits; see norm_fp8.cu.
int b200_rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldres, void* h_out, const void* w, void* q, float* scale, long long T,
                     int H, float eps, int group, void* stream);

// Tokens sorted by expert and back; see moe_sort.cu.
int b200_expert_order(const void* idx, int idx64, long long n, int experts, int* row_of, int* offsets, void* stream);
int b200_permute_rows(const void* x, long long pitch, void* rows, const int* row_of, const float* scale, float* row_scale, int groups, long long tokens,
                      int k, long long row_bytes, int elem, void* stream);
int b200_unpermute_rows(const void* rows, long long pitch, const float* w, const int* row_of, void* out, long long tokens, int k, int H, int fp32,
                        void* stream);
int b200_unpermute_rows_bwd(const void* dout, const void* rows, long long pitch, const float* w, const int* row_of, void* drows, float* dw,
                            long long tokens, int k, int H, int fp32, void* stream);

// One tensor of an AdamW step: p and g are bf16 unless the flags say otherwise; m and v are e4m3 codes with a scale for every 256 elements, or fp32;
// master is null, or an fp32 copy of a bf16 p. keep = 1 - lr * weight_decay.
struct B200AdamwTensor {
  void *p, *g, *m, *v;
  float *m_scale, *v_scale, *master;
  long long n;
  float keep;
  unsigned char p_fp32, g_fp32;
};
// *launches (unless null): kernels launched; see adamw_many.cu.
int b200_adamw_many(const B200AdamwTensor* list, int count, int bits, double lr, double beta1, double beta2, double eps, long long step, double grad_scale,
                    int zero_grad, int* launches, void* stream);

// Activations in 8 bits, codes [rows][width] and a byte for every 32 of a row (or what is left of it), and SwiGLU with gate and up kept so, as rows 2t and
// 2t + 1 of F; see kept8.cu. width and F are multiples of 8. swiglu_kept8 makes gate|up of what is kept, and act unless that is null.
int b200_keep8(const void* x, long long pitch, void* codes, void* powers, long long rows, int width, void* stream);
int b200_kept8(const void* codes, const void* powers, void* x, long long rows, int width, void* stream);
int b200_swiglu_keep8(const void* gu, void* act, void* codes, void* powers, long long T, int F, void* stream);
int b200_swiglu_bwd8(const void* dout, const void* codes, const void* powers, void* dgu, long long T, int F, void* stream);
int b200_swiglu_kept8(const void* codes, const void* powers, void* gu, void* act, long long T, int F, void* stream);

// Attention with a window and sinks, and its gradients; see attention.cu. Tensors are [batch][token][head][hd] bf16 with element strides (multiples of
// eight; any for a dimension of one) and contiguous heads; out, dq, dk and dv are contiguous. lse and delta are [B][nq][S rounded up to 128] floats.
// dq, or dk and dv together, may be null; sums are b200_attention_bwd_workspace's number of floats.
struct B200AttnTensor {
  const void* data;
  long long batch, token, head;
};
struct B200AttnArgs {
  B200AttnTensor q, k, v, dout;
  void *out, *rest;   // rest: null, or a byte for each element of out, written beside it and read for delta
  float *lse, *delta, *sums;
  void *dq, *dk, *dv;
  const int* lengths;   // [B] or null
  int B, S, nq, nkv, hd, window, sinks;
  float scale;
};
int b200_attention_fwd(const B200AttnArgs* args, void* stream);
long long b200_attention_bwd_workspace(const B200AttnArgs* args);
int b200_attention_bwd(const B200AttnArgs* args, int* launches, void* stream);

}  // extern "C"

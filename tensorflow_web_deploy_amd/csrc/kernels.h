// Host-side launch API for the CDNA4 HIP kernels (bound in bindings.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

// gemm_conv.hip — C = act(A @ B^T + bias [+ residual]), bf16 in/out, f32 acc
int splitk_plan(int M, int N, int K);
// act: 0 none, 1 relu, 5 gelu; ldc: C row stride (0 = N)
void launch_gemm_bf16(const void* A, const void* B, void* C,
                      const float* bias, const void* residual, int M, int N,
                      int K, int Kp, int64_t a_bytes, int act,
                      hipStream_t stream, float* ws = nullptr,
                      int splitk = 1, int ldc = 0);
bool launch_conv_direct(const void* X, const void* W2, void* Y,
                        const float* bias, int Nimg, int H, int W, int C,
                        int R, int S, int Cout, int sh, int sw, int pt,
                        int pl, int HO, int WO, int Kp, int act,
                        hipStream_t stream, int ldc);
void launch_conv2d_bf16(const void* X, const void* B, void* C,
                        const float* bias, const void* residual, int Nimg,
                        int H, int W, int Cin, int R, int S, int Cout, int sh,
                        int sw, int pt, int pl, int HO, int WO, int Kp,
                        int act, hipStream_t stream, float* ws = nullptr,
                        int splitk = 1, int ldc = 0);

void launch_dwconv_bf16(const void* x, const void* w, const float* bias,
                        const void* residual, void* y, int N, int H,
                        int W, int C, int HO, int WO, int R, int S,
                        int sh, int sw, int pt, int pl, int act,
                        hipStream_t stream);

void launch_jpeg_decode(void* arena, void* planes, const void* flags,
                        int n, int64_t slot_bytes, hipStream_t stream);

void launch_gemm_8p(const void* A, const void* B, void* C,
                    const float* bias, const void* residual, int M,
                    int N, int K, int Kp, int act, int ldc,
                    hipStream_t stream);

// pool_reduce.hip
void launch_maxpool_bf16(const void* X, void* Y, int Nimg, int H, int W,
                         int C, int kh, int kw, int sh, int sw, int pt,
                         int pl, int HO, int WO, hipStream_t stream);
void launch_avgpool_bf16(const void* X, void* Y, int Nimg, int H, int W,
                         int C, int kh, int kw, int sh, int sw, int pt,
                         int pl, int HO, int WO, hipStream_t stream);
void launch_global_mean_bf16(const void* X, void* Y, int Nimg, int HW, int C,
                             hipStream_t stream);
void launch_softmax_bf16(const void* X, float* Y, int M, int N,
                         hipStream_t stream);
void launch_softmax_bf16_out(const void* X, void* Y, int M, int N,
                             hipStream_t stream);

// layernorm.hip
void launch_layernorm_bf16(const void* X, const float* gamma,
                           const float* beta, void* Y, int64_t rows, int C,
                           float eps, hipStream_t stream);

// fully-strided batched GEMM: C[b1,b2] = A[b1,b2] @ B[b1,b2]^T with
// independent row strides (lda/ldb/ldc) and 2D batch strides — lets
// attention run directly on [N, tokens, heads, dim] views (no transposes)
void launch_gemm_strided_bf16(const void* A, const void* B, void* C,
                              int batch1, int batch2, int M, int N, int K,
                              int lda, int ldb, int ldc, int64_t sA1,
                              int64_t sA2, int64_t sB1, int64_t sB2,
                              int64_t sC1, int64_t sC2, int64_t a_total,
                              hipStream_t stream);

// gemm_conv.hip (strided-batch, MODE 0, no epilogue fusion)
void launch_gemm_batched_bf16(const void* A, const void* B, void* C,
                              int batch, int M, int N, int K, int Kp,
                              int64_t sA, int64_t sB, int64_t sC,
                              hipStream_t stream);

// elementwise.hip
void launch_cast_f32_bf16(const float* X, void* Y, int64_t n,
                          hipStream_t stream);
void launch_cast_bf16_f32(const void* X, float* Y, int64_t n,
                          hipStream_t stream);
void launch_cast_f32_pad_bf16(const float* X, void* Y, int64_t rows,
                              int Cin, int Cpad, hipStream_t stream);
void launch_channel_pad_bf16(const void* X, void* Y, int64_t rows, int Cin,
                             int Cpad, hipStream_t stream);
void launch_add_relu_bf16(const void* A, const void* B, void* Y, int64_t n,
                          bool relu, hipStream_t stream);
void launch_bias_act_bf16(const void* X, const float* bias, void* Y,
                          int64_t rows, int C, int act, hipStream_t stream);
void launch_scale_shift_bf16(const void* X, const float* scale,
                             const float* shift, void* Y, int64_t rows, int C,
                             bool relu, hipStream_t stream);

// preprocess.hip
void launch_resize_norm(const void* src, int sh, int sw, int sc, float* dst,
                        int dh, int dw, int dc, int norm,
                        hipStream_t stream);
void launch_resize_norm_batch(const void* arena, const int* meta,
                              float* dst, int n, int dh, int dw, int dc,
                              int norm, hipStream_t stream);

// attn_fused.hip — fused softmax attention (S <= 256, D = 64)
void launch_attn_fused_bf16(const void* Q, const void* K, const void* V,
                            void* O, int batch1, int batch2, int S,
                            int64_t sQ1, int64_t sQ2, int lqd, int64_t sK1,
                            int64_t sK2, int lkd, int64_t sV1, int64_t sV2,
                            int lvd, int64_t sO1, int64_t sO2, int lod,
                            float scale, hipStream_t stream);

// gemm_fp8.hip — e4m3 with a scale for each 128 values along K.
// X [M][K] (row stride ldx) bf16 or f32 -> Q [M][Kp], Kp = K up to whole
// blocks; S [Kp/128][M] (block_rows 1) or [M/128][Kp/128] (block_rows 128)
void launch_quant_fp8(const void* X, bool f32, int64_t ldx, int64_t M, int K,
                      void* Q, int Kp, float* S, int block_rows,
                      hipStream_t stream);
// floats that launch_gemm_fp8 needs at `part`
int64_t gemm_fp8_workspace(int M, int N, int Kp, bool f32);
// C = act(A @ B^T + bias + residual), C bf16 or f32 with row stride ldc; act:
// 0 none, 1 relu, 2 relu6, 5 gelu
void launch_gemm_fp8(const void* A, const float* SA, const void* B,
                     const float* SB, void* C, bool f32, int64_t ldc,
                     const float* bias, const void* residual, int64_t ldr,
                     int M, int N, int Kp, int act, float* part,
                     hipStream_t stream);

// moe.hip — mixture-of-experts layers
// Y [T][E] f32 = X [T][D] (row stride ldx) W^T, X bf16; W [3][E][D up to 64s]
// bf16: the three add up to the weights. E <= 512
void launch_moe_logits(const void* X, int64_t ldx, const void* W, float* Y,
                       int T, int D, int E, hipStream_t stream);
// logits [T][E] (row stride ldx) bf16 or f32 -> the k experts of each row and
// their weights; rows or experts that have none get id -1 and weight 0.
// E <= 512, k <= 64, groups <= 64
void launch_moe_route(const void* X, bool f32, int64_t ldx, const float* bias,
                      int* ids, float* weights, int T, int E, int k,
                      bool sigmoid, int groups, int kept, int best,
                      bool renorm, float scale, hipStream_t stream);
// Y[t] = residual[t] + sum_j weights[t][j] mlp_{ids[t][j]}(X[t]); ids outside
// of 0..E-1 name no expert. Weights are bf16 [E][H][D up to 64s] and
// [E][D][H up to 64s], or e4m3, up to 128s, with their scales.
struct MoeMlp {
  const void *X, *W1, *W2, *residual;
  const int* ids;
  const float *weights, *S1, *b1, *S2, *b2;
  void* Y;
  int64_t ldx, ldy, ldr;
  int T, E, k, D, H, act;
  bool fp8;
};
int64_t moe_mlp_workspace(const MoeMlp& m);  // bytes
void launch_moe_mlp(const MoeMlp& m, void* ws, hipStream_t stream);

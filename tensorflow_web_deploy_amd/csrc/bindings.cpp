// pybind11/torch bindings for the CDNA4 HIP kernels (native path of the
// engine). Pure HIP — no CUDA compatibility layer: streams come from
// c10::hip directly.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <cmath>

#include "kernels.h"

namespace {

hipStream_t cur_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

void check_bf16(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// 2D output that may be a column-slice view: [M][N] with row stride ldc
int check_out2d(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == 2 && t.stride(1) == 1, name,
              " must be 2D with contiguous rows");
  return (int)t.stride(0);
}

// C[M][N] = act(A[M][K] @ B[N][K]^T + bias [+ residual])
void gemm_bf16(torch::Tensor A, torch::Tensor B, torch::Tensor C,
               c10::optional<torch::Tensor> bias,
               c10::optional<torch::Tensor> residual, int64_t K,
               int64_t act) {
  check_bf16(A, "A");
  check_bf16(B, "B");
  int ldc = check_out2d(C, "C");
  int64_t M = C.size(0), N = C.size(1);
  int64_t Kp = B.size(1);
  TORCH_CHECK(B.size(0) >= N, "B rows < N");
  TORCH_CHECK(K % 8 == 0, "K must be a multiple of 8");
  const float* bptr = nullptr;
  if (bias) {
    TORCH_CHECK(bias->scalar_type() == torch::kFloat32, "bias must be f32");
    bptr = bias->data_ptr<float>();
  }
  const void* rptr = nullptr;
  if (residual) {
    check_bf16(*residual, "residual");
    rptr = residual->data_ptr();
  }
  int sk = ldc == (int)N ? splitk_plan((int)M, (int)N, (int)K) : 1;
  torch::Tensor ws;
  float* wptr = nullptr;
  if (sk > 1) {
    ws = torch::empty({(int64_t)sk * M * N},
                      torch::dtype(torch::kFloat32).device(A.device()));
    wptr = ws.data_ptr<float>();
  }
  launch_gemm_bf16(A.data_ptr(), B.data_ptr(), C.data_ptr(), bptr, rptr,
                   (int)M, (int)N, (int)K, (int)Kp,
                   A.numel() * 2, (int)act, cur_stream(), wptr, sk, ldc);
}

// X [N,H,W,C] bf16, W2 [Cout][Kp] (pre-transposed HWIO, K-padded)
void conv2d_bf16(torch::Tensor X, torch::Tensor W2, torch::Tensor Y,
                 c10::optional<torch::Tensor> bias,
                 c10::optional<torch::Tensor> residual, int64_t R, int64_t S,
                 int64_t sh, int64_t sw, int64_t pt, int64_t pl,
                 int64_t act) {
  check_bf16(X, "X");
  check_bf16(W2, "W");
  TORCH_CHECK(X.dim() == 4 && Y.dim() == 4);
  // Y may be a channel-slice of a concat buffer: last dim contiguous,
  // pixel stride = total concat channels
  TORCH_CHECK(Y.is_cuda() && Y.scalar_type() == torch::kBFloat16);
  TORCH_CHECK(Y.stride(3) == 1);
  int ldc = (int)Y.stride(2);
  int Nimg = X.size(0), H = X.size(1), W = X.size(2), Cin = X.size(3);
  int HO = Y.size(1), WO = Y.size(2), Cout = Y.size(3);
  TORCH_CHECK(Cin % 8 == 0, "Cin must be a multiple of 8 (pad first)");
  const float* bptr = nullptr;
  if (bias) bptr = bias->data_ptr<float>();
  const void* rptr = nullptr;
  if (residual) {
    check_bf16(*residual, "residual");
    rptr = residual->data_ptr();
  }
  int M = Nimg * HO * WO;
  int K = (int)(R * S) * Cin;
  int sk = ldc == Cout ? splitk_plan(M, Cout, K) : 1;
  torch::Tensor ws;
  float* wptr = nullptr;
  if (sk > 1) {
    ws = torch::empty({(int64_t)sk * M * Cout},
                      torch::dtype(torch::kFloat32).device(X.device()));
    wptr = ws.data_ptr<float>();
  }
  launch_conv2d_bf16(X.data_ptr(), W2.data_ptr(), Y.data_ptr(), bptr, rptr,
                     Nimg, H, W, Cin, (int)R, (int)S, Cout, (int)sh, (int)sw,
                     (int)pt, (int)pl, HO, WO, (int)W2.size(1), (int)act,
                     cur_stream(), wptr, sk, ldc);
}

void maxpool_bf16(torch::Tensor X, torch::Tensor Y, int64_t kh, int64_t kw,
                  int64_t sh, int64_t sw, int64_t pt, int64_t pl) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  launch_maxpool_bf16(X.data_ptr(), Y.data_ptr(), X.size(0), X.size(1),
                      X.size(2), X.size(3), kh, kw, sh, sw, pt, pl, Y.size(1),
                      Y.size(2), cur_stream());
}

void avgpool_bf16(torch::Tensor X, torch::Tensor Y, int64_t kh, int64_t kw,
                  int64_t sh, int64_t sw, int64_t pt, int64_t pl) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  launch_avgpool_bf16(X.data_ptr(), Y.data_ptr(), X.size(0), X.size(1),
                      X.size(2), X.size(3), kh, kw, sh, sw, pt, pl, Y.size(1),
                      Y.size(2), cur_stream());
}

void global_mean_bf16(torch::Tensor X, torch::Tensor Y) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  launch_global_mean_bf16(X.data_ptr(), Y.data_ptr(), X.size(0),
                          X.size(1) * X.size(2), X.size(3), cur_stream());
}

void softmax_bf16(torch::Tensor X, torch::Tensor Y) {
  check_bf16(X, "X");
  TORCH_CHECK(Y.scalar_type() == torch::kFloat32);
  launch_softmax_bf16(X.data_ptr(), Y.data_ptr<float>(), X.size(0), X.size(1),
                      cur_stream());
}

void softmax_bf16_out(torch::Tensor X, torch::Tensor Y) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  launch_softmax_bf16_out(X.data_ptr(), Y.data_ptr(), X.size(0), X.size(1),
                          cur_stream());
}

void cast_f32_bf16(torch::Tensor X, torch::Tensor Y) {
  TORCH_CHECK(X.scalar_type() == torch::kFloat32 && X.is_contiguous());
  check_bf16(Y, "Y");
  launch_cast_f32_bf16(X.data_ptr<float>(), Y.data_ptr(), X.numel(),
                       cur_stream());
}

void cast_bf16_f32(torch::Tensor X, torch::Tensor Y) {
  check_bf16(X, "X");
  TORCH_CHECK(Y.scalar_type() == torch::kFloat32);
  launch_cast_bf16_f32(X.data_ptr(), Y.data_ptr<float>(), X.numel(),
                       cur_stream());
}

void cast_f32_pad_bf16(torch::Tensor X, torch::Tensor Y) {
  TORCH_CHECK(X.scalar_type() == torch::kFloat32 && X.is_contiguous());
  check_bf16(Y, "Y");
  int64_t rows = X.numel() / X.size(-1);
  launch_cast_f32_pad_bf16(X.data_ptr<float>(), Y.data_ptr(), rows,
                           X.size(-1), Y.size(-1), cur_stream());
}

void channel_pad_bf16(torch::Tensor X, torch::Tensor Y) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  int64_t rows = X.numel() / X.size(-1);
  launch_channel_pad_bf16(X.data_ptr(), Y.data_ptr(), rows, X.size(-1),
                          Y.size(-1), cur_stream());
}

void add_relu_bf16(torch::Tensor A, torch::Tensor B, torch::Tensor Y,
                   bool relu) {
  check_bf16(A, "A");
  check_bf16(B, "B");
  check_bf16(Y, "Y");
  launch_add_relu_bf16(A.data_ptr(), B.data_ptr(), Y.data_ptr(), A.numel(),
                       relu, cur_stream());
}

void bias_act_bf16(torch::Tensor X, c10::optional<torch::Tensor> bias,
                   torch::Tensor Y, int64_t act) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  int C = X.size(-1);
  const float* bptr = nullptr;
  if (bias) {
    TORCH_CHECK(bias->numel() == C, "bias size ", bias->numel(),
                " != channels ", C);
    bptr = bias->data_ptr<float>();
  }
  launch_bias_act_bf16(X.data_ptr(), bptr, Y.data_ptr(), X.numel() / C, C,
                       (int)act, cur_stream());
}

void scale_shift_bf16(torch::Tensor X, torch::Tensor scale,
                      torch::Tensor shift, torch::Tensor Y, bool relu) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  int C = X.size(-1);
  TORCH_CHECK(scale.numel() == C && shift.numel() == C,
              "scale/shift size mismatch vs channels ", C);
  launch_scale_shift_bf16(X.data_ptr(), scale.data_ptr<float>(),
                          shift.data_ptr<float>(), Y.data_ptr(),
                          X.numel() / C, C, relu, cur_stream());
}

void layernorm_bf16(torch::Tensor X, c10::optional<torch::Tensor> gamma,
                    c10::optional<torch::Tensor> beta, torch::Tensor Y,
                    double eps) {
  check_bf16(X, "X");
  check_bf16(Y, "Y");
  int C = X.size(-1);
  TORCH_CHECK(C % 8 == 0 && C <= 2048, "layernorm C must be %8 and <=2048");
  const float* g = gamma ? gamma->data_ptr<float>() : nullptr;
  const float* b = beta ? beta->data_ptr<float>() : nullptr;
  launch_layernorm_bf16(X.data_ptr(), g, b, Y.data_ptr(), X.numel() / C, C,
                        (float)eps, cur_stream());
}

// batched C[b] = A[b] @ B[b]^T  (A [batch,M,K], B [batch,N,K], C [batch,M,N])
void gemm_batched_bf16(torch::Tensor A, torch::Tensor B, torch::Tensor C) {
  check_bf16(A, "A");
  check_bf16(B, "B");
  check_bf16(C, "C");
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && C.dim() == 3);
  int batch = A.size(0), M = A.size(1), K = A.size(2);
  int N = B.size(1);
  TORCH_CHECK(B.size(0) == batch && C.size(0) == batch);
  TORCH_CHECK(B.size(2) == K && C.size(1) == M && C.size(2) == N);
  TORCH_CHECK(K % 8 == 0, "batched gemm K must be a multiple of 8");
  launch_gemm_batched_bf16(A.data_ptr(), B.data_ptr(), C.data_ptr(), batch,
                           M, N, K, K, (int64_t)M * K, (int64_t)N * K,
                           (int64_t)M * N, cur_stream());
}

// src: uint8 [sh, sw, sc]; dst: f32 [dh, dw, dc] on the given stream
void resize_norm(torch::Tensor src, torch::Tensor dst, int64_t norm) {
  TORCH_CHECK(src.is_cuda() && src.scalar_type() == torch::kUInt8
              && src.is_contiguous());
  TORCH_CHECK(dst.is_cuda() && dst.scalar_type() == torch::kFloat32
              && dst.is_contiguous());
  launch_resize_norm(src.data_ptr(), src.size(0), src.size(1), src.size(2),
                     dst.data_ptr<float>(), dst.size(0), dst.size(1),
                     dst.size(2), (int)norm, cur_stream());
}

// arena u8 (packed images), meta i32 [n,4] = {off, sh, sw, sc} on GPU,
// dst f32 [n, H, W, C]
void resize_norm_batch(torch::Tensor arena, torch::Tensor meta,
                       torch::Tensor dst, int64_t norm) {
  TORCH_CHECK(arena.is_cuda() && arena.scalar_type() == torch::kUInt8);
  TORCH_CHECK(meta.is_cuda() && meta.scalar_type() == torch::kInt32);
  TORCH_CHECK(dst.is_cuda() && dst.scalar_type() == torch::kFloat32
              && dst.is_contiguous());
  launch_resize_norm_batch(arena.data_ptr(), meta.data_ptr<int>(),
                           dst.data_ptr<float>(), dst.size(0), dst.size(1),
                           dst.size(2), dst.size(3), (int)norm,
                           cur_stream());
}

// Attention GEMM on 4D views: every tensor supplies its own strides.
// A: [B1, M, ...] with k contiguous; B: [B1, N-rows ...]; C likewise.
// Python passes logical dims + strides explicitly (views, zero-copy).
void gemm_strided_bf16(torch::Tensor A, torch::Tensor B, torch::Tensor C,
                       int64_t batch1, int64_t batch2, int64_t M, int64_t N,
                       int64_t K, int64_t lda, int64_t ldb, int64_t ldc,
                       int64_t sA1, int64_t sA2, int64_t sB1, int64_t sB2,
                       int64_t sC1, int64_t sC2) {
  TORCH_CHECK(A.is_cuda() && A.scalar_type() == torch::kBFloat16);
  TORCH_CHECK(B.is_cuda() && B.scalar_type() == torch::kBFloat16);
  TORCH_CHECK(C.is_cuda() && C.scalar_type() == torch::kBFloat16);
  TORCH_CHECK(K % 8 == 0, "strided gemm K must be %8");
  launch_gemm_strided_bf16(A.data_ptr(), B.data_ptr(), C.data_ptr(),
                           (int)batch1, (int)batch2, (int)M, (int)N, (int)K,
                           (int)lda, (int)ldb, (int)ldc, sA1, sA2, sB1, sB2,
                           sC1, sC2, A.numel(), cur_stream());
}

// Fused attention: Q/K/V/O are 4D views [B1, S, B2, D] or [B1, B2, S, D]
// etc — every tensor supplies explicit strides; D must be 64, S <= 256.
void attn_fused_bf16(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                     torch::Tensor O, int64_t batch1, int64_t batch2,
                     int64_t S, int64_t sQ1, int64_t sQ2, int64_t lqd,
                     int64_t sK1, int64_t sK2, int64_t lkd, int64_t sV1,
                     int64_t sV2, int64_t lvd, int64_t sO1, int64_t sO2,
                     int64_t lod, double scale) {
  TORCH_CHECK(Q.is_cuda() && Q.scalar_type() == torch::kBFloat16);
  TORCH_CHECK(S <= 256, "fused attention supports S <= 256");
  launch_attn_fused_bf16(Q.data_ptr(), K.data_ptr(), V.data_ptr(),
                         O.data_ptr(), (int)batch1, (int)batch2, (int)S,
                         sQ1, sQ2, (int)lqd, sK1, sK2, (int)lkd, sV1, sV2,
                         (int)lvd, sO1, sO2, (int)lod, (float)scale,
                         cur_stream());
}

// ---- fp8 dense layers. Types and shapes are looked at before the device,
// so that a wrong call is named wherever it is made.

constexpr auto kFp8 = c10::ScalarType::Float8_e4m3fn;

void check_type(const torch::Tensor& t, c10::ScalarType type,
                const char* name) {
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ",
              t.scalar_type());
}

void check_shape(const torch::Tensor& t, c10::IntArrayRef shape,
                 const char* name) {
  TORCH_CHECK(t.sizes() == shape, name, " must be ", shape, ", got ",
              t.sizes());
}

void check_whole(const torch::Tensor& t, c10::ScalarType type,
                 c10::IntArrayRef shape, const char* name) {
  check_type(t, type, name);
  check_shape(t, shape, name);
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// the kernels take these 16 bytes at a time
void check_aligned(const torch::Tensor& t, const char* name) {
  TORCH_CHECK((uintptr_t)t.data_ptr() % 16 == 0, name,
              " must start at a multiple of 16 bytes");
}

// rows of contiguous values that may lie apart, but not over each other
void check_rows(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2D");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name,
              " must have contiguous rows");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name,
              " must have rows that don't overlap");
}

int64_t row_stride(const torch::Tensor& t) {
  return t.size(0) <= 1 ? t.size(1) : t.stride(0);
}

void check_bf16_or_f32(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16 ||
                  t.scalar_type() == torch::kFloat32,
              name, " must be bf16 or f32, got ", t.scalar_type());
}

void check_act(int64_t act) {
  TORCH_CHECK(act == 0 || act == 1 || act == 2 || act == 5,
              "act must be 0 (none), 1 (relu), 2 (relu6) or 5 (gelu), got ",
              act);
}

// Whether two tensors, each whole or rows that may lie apart, share a byte.
// Rows of one width apart from each other may lie beside those of the other.
bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  if (!a.numel() || !b.numel() || a.is_meta() || b.is_meta()) return false;
  auto rows = [](const torch::Tensor& t) {
    return t.dim() == 2 && t.size(0) > 1;
  };
  auto width = [&](const torch::Tensor& t) {
    return (rows(t) ? t.size(1) : t.numel()) * (int64_t)t.element_size();
  };
  auto apart = [&](const torch::Tensor& t) {
    return rows(t) ? t.stride(0) * (int64_t)t.element_size() : 0;
  };
  auto end = [&](const torch::Tensor& t) {
    return (uintptr_t)t.data_ptr() +
           (rows(t) ? (t.size(0) - 1) * apart(t) : 0) + width(t);
  };
  const auto pa = (uintptr_t)a.data_ptr(), pb = (uintptr_t)b.data_ptr();
  if (pa >= end(b) || pb >= end(a)) return false;
  const int64_t step = apart(a);
  if (step == 0 || step != apart(b)) return true;
  const int64_t d = ((int64_t)(pb - pa) % step + step) % step;
  return d < width(a) || step - d < width(b);
}

bool same_place(const torch::Tensor& a, const torch::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.scalar_type() == b.scalar_type() &&
         a.sizes() == b.sizes() &&
         (a.size(0) <= 1 || a.stride(0) == b.stride(0));
}

// what is written first, then what it may not lie over
void check_apart(c10::ArrayRef<std::pair<const torch::Tensor*, const char*>>
                     tensors) {
  for (auto& [t, name] : tensors.slice(1))
    TORCH_CHECK(!overlap(*tensors[0].first, *t), tensors[0].second,
                " must not overlap ", name);
}

// all of them on one GPU, which the launches then go to
void check_devices(c10::ArrayRef<std::pair<const torch::Tensor*, const char*>>
                       tensors) {
  const torch::Tensor& first = *tensors[0].first;
  for (auto& [t, name] : tensors) {
    TORCH_CHECK(t->is_cuda(), name, " must be on GPU");
    TORCH_CHECK(t->device() == first.device(), name, " is on ", t->device(),
                ", ", tensors[0].second, " on ", first.device());
  }
}

// a launch holds fewer than 2^32 threads along x: with 16 rows, or a tile of
// 128 x 128, to a workgroup of 256, or 16 columns to one of 512
constexpr int64_t kMaxRows = 1 << 27, kMaxTiles = 1 << 24;
constexpr int64_t kMaxColumns = (1 << 27) - 16;

int64_t blocks128(int64_t n) { return (n + 127) / 128; }

// X [M,K] bf16|f32 -> Q [M,Kp] e4m3, Kp = K up to whole blocks of 128 (the
// rest 0), and the scales: block_rows 1 (activations): S [Kp/128, M], one for
// each row and 128 of K; block_rows 128 (weights): S [ceil(M/128), Kp/128]
void quant_fp8(torch::Tensor X, torch::Tensor Q, torch::Tensor S,
               int64_t block_rows) {
  check_bf16_or_f32(X, "X");
  check_rows(X, "X");
  TORCH_CHECK(block_rows == 1 || block_rows == 128,
              "block_rows must be 1 or 128, got ", block_rows);
  const int64_t M = X.size(0), K = X.size(1), Kb = blocks128(K);
  TORCH_CHECK(K >= 1 && K <= 1 << 22, "K must be 1 to 2^22, got ", K);
  TORCH_CHECK(M < kMaxRows && blocks128(M) * Kb < kMaxTiles,
              "X is too large: ", X.sizes());
  check_whole(Q, kFp8, {M, Kb * 128}, "Q");
  check_aligned(Q, "Q");
  if (block_rows == 1)
    check_whole(S, torch::kFloat32, {Kb, M}, "S");
  else
    check_whole(S, torch::kFloat32, {blocks128(M), Kb}, "S");
  check_apart({{&Q, "Q"}, {&X, "X"}});
  check_apart({{&S, "S"}, {&X, "X"}, {&Q, "Q"}});
  check_devices({{&X, "X"}, {&Q, "Q"}, {&S, "S"}});
  if (M == 0) return;
  const c10::DeviceGuard guard(X.device());
  launch_quant_fp8(X.data_ptr(), X.scalar_type() == torch::kFloat32,
                   row_stride(X), M, (int)K, Q.data_ptr(), (int)Kb * 128,
                   S.data_ptr<float>(), (int)block_rows, cur_stream());
}

// C[M][N] = act(A @ B^T + bias + residual), C bf16 or f32, residual bf16. A
// [M,Kp] with SA [Kp/128, M], B [N,Kp] with SB [ceil(N/128), Kp/128]: as
// quant_fp8 leaves them with block_rows 1 and 128
void gemm_fp8(torch::Tensor A, torch::Tensor SA, torch::Tensor B,
              torch::Tensor SB, torch::Tensor C,
              c10::optional<torch::Tensor> bias,
              c10::optional<torch::Tensor> residual, int64_t act) {
  const bool f32 = C.scalar_type() == torch::kFloat32;
  TORCH_CHECK(C.scalar_type() == torch::kBFloat16 || (f32 && C.is_cuda()),
              "C must be BFloat16 or, on a GPU, Float, got ", C.scalar_type(),
              " on ", C.device());
  check_rows(C, "C");
  check_type(A, kFp8, "A");
  TORCH_CHECK(A.dim() == 2, "A must be 2D");
  const int64_t M = C.size(0), N = C.size(1), Kp = A.size(1);
  TORCH_CHECK(Kp >= 128 && Kp % 128 == 0 && Kp <= 1 << 22,
              "A must hold whole blocks of 128 along K, 2^22 values at most, "
              "got ", Kp);
  TORCH_CHECK(N >= 1 && N <= kMaxColumns && M < kMaxRows &&
                  blocks128(M) * blocks128(N) < kMaxTiles,
              "C is too large or has no columns: ", C.sizes());
  TORCH_CHECK(M * (Kp / 128) < 1 << 30, "SA is too large");
  check_whole(A, kFp8, {M, Kp}, "A");
  check_whole(SA, torch::kFloat32, {Kp / 128, M}, "SA");
  check_whole(B, kFp8, {N, Kp}, "B");
  check_aligned(A, "A");
  check_aligned(B, "B");
  check_whole(SB, torch::kFloat32, {blocks128(N), Kp / 128}, "SB");
  check_act(act);
  std::vector<std::pair<const torch::Tensor*, const char*>> all = {
      {&A, "A"}, {&SA, "SA"}, {&B, "B"}, {&SB, "SB"}, {&C, "C"}};
  if (bias) {
    check_whole(*bias, torch::kFloat32, {N}, "bias");
    all.push_back({&*bias, "bias"});
  }
  if (residual) {
    check_type(*residual, torch::kBFloat16, "residual");
    check_shape(*residual, {M, N}, "residual");
    check_rows(*residual, "residual");
    all.push_back({&*residual, "residual"});
  }
  check_apart({{&C, "C"}, {&A, "A"}, {&SA, "SA"}, {&B, "B"}, {&SB, "SB"}});
  if (bias) check_apart({{&C, "C"}, {&*bias, "bias"}});
  if (residual && !same_place(C, *residual))
    check_apart({{&C, "C"}, {&*residual, "residual"}});
  check_devices(all);
  if (M == 0) return;
  const c10::DeviceGuard guard(A.device());
  const int64_t floats = gemm_fp8_workspace((int)M, (int)N, (int)Kp, f32);
  torch::Tensor ws;
  if (floats) ws = torch::empty({floats}, SA.options());
  launch_gemm_fp8(A.data_ptr(), SA.data_ptr<float>(), B.data_ptr(),
                  SB.data_ptr<float>(), C.data_ptr(), f32, row_stride(C),
                  bias ? bias->data_ptr<float>() : nullptr,
                  residual ? residual->data_ptr() : nullptr,
                  residual ? row_stride(*residual) : 0, (int)M, (int)N,
                  (int)Kp, (int)act, floats ? ws.data_ptr<float>() : nullptr,
                  cur_stream());
}

// ---- mixture-of-experts layers

// logits [T,E] f32 = X [T,D] bf16 @ W^T. W [3,E,D up to 64s] bf16, filled up
// with zeros: its three parts add up to the f32 weights, each the rounding of
// what those before it leave
void moe_logits(torch::Tensor X, torch::Tensor W, torch::Tensor logits) {
  check_type(X, torch::kBFloat16, "X");
  check_rows(X, "X");
  const int64_t T = X.size(0), D = X.size(1);
  TORCH_CHECK(T < kMaxRows, "too many rows: ", T);
  TORCH_CHECK(D >= 1 && D <= 1 << 18, "width must be 1 to 2^18, got ", D);
  TORCH_CHECK(W.dim() == 3, "W must be 3D");
  const int64_t E = W.size(1);
  TORCH_CHECK(E >= 1 && E <= 512, "1 to 512 experts, got ", E);
  // 128 rows and 32 experts to a workgroup of 512 threads
  TORCH_CHECK((T + 127) / 128 * ((E + 31) / 32) < 1 << 23,
              "too many rows: ", T);
  check_whole(W, torch::kBFloat16, {3, E, (D + 63) / 64 * 64}, "W");
  check_aligned(W, "W");
  check_whole(logits, torch::kFloat32, {T, E}, "logits");
  check_apart({{&logits, "logits"}, {&X, "X"}, {&W, "W"}});
  check_devices({{&X, "X"}, {&W, "W"}, {&logits, "logits"}});
  if (T == 0) return;
  const c10::DeviceGuard guard(X.device());
  launch_moe_logits(X.data_ptr(), row_stride(X), W.data_ptr(),
                    logits.data_ptr<float>(), (int)T, (int)D, (int)E,
                    cur_stream());
}

// logits [T,E] bf16|f32 -> ids i32 [T,k], weights f32 [T,k]. score: 0 softmax,
// 1 sigmoid; bias f32 [E] is added for the choice alone. With groups > 1 the
// experts are taken from the `kept` groups whose `best` (1 or 2) largest
// score + bias add up to the most. A logit of -inf or NaN shuts an expert for
// its row; places that no expert is left for get id -1 and weight 0. Choices
// are those of the scores in 64 bits, the lower index first among equals.
void moe_route(torch::Tensor logits, c10::optional<torch::Tensor> bias,
               torch::Tensor ids, torch::Tensor weights, int64_t score,
               int64_t groups, int64_t kept, int64_t best, bool renorm,
               double scale) {
  check_bf16_or_f32(logits, "logits");
  check_rows(logits, "logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= 512, "1 to 512 experts, got ", E);
  TORCH_CHECK(T < kMaxRows, "too many rows: ", T);
  TORCH_CHECK(score == 0 || score == 1,
              "score must be 0 (softmax) or 1 (sigmoid), got ", score);
  TORCH_CHECK(groups >= 1 && groups <= 64 && E % groups == 0,
              "groups must be 1 to 64 and divide the experts, got ", groups);
  TORCH_CHECK(kept >= 1 && kept <= groups, "kept must be 1 to groups, got ",
              kept);
  TORCH_CHECK(best == 1 || best == 2, "best must be 1 or 2, got ", best);
  TORCH_CHECK(std::isfinite((float)scale), "scale must be finite in f32, got ",
              scale);
  TORCH_CHECK(ids.dim() == 2, "ids must be 2D");
  const int64_t k = ids.size(1);
  TORCH_CHECK(k >= 1 && k <= 64 && k <= kept * (E / groups),
              "k must be 1 to 64 and no more than the kept groups hold, got ",
              k);
  check_whole(ids, torch::kInt32, {T, k}, "ids");
  check_whole(weights, torch::kFloat32, {T, k}, "weights");
  std::vector<std::pair<const torch::Tensor*, const char*>> all = {
      {&logits, "logits"}, {&ids, "ids"}, {&weights, "weights"}};
  if (bias) {
    check_whole(*bias, torch::kFloat32, {E}, "bias");
    all.push_back({&*bias, "bias"});
    check_apart({{&ids, "ids"}, {&*bias, "bias"}});
    check_apart({{&weights, "weights"}, {&*bias, "bias"}});
  }
  check_apart({{&ids, "ids"}, {&logits, "logits"}});
  check_apart({{&weights, "weights"}, {&logits, "logits"}, {&ids, "ids"}});
  check_devices(all);
  if (T == 0) return;
  const c10::DeviceGuard guard(logits.device());
  launch_moe_route(logits.data_ptr(),
                   logits.scalar_type() == torch::kFloat32,
                   row_stride(logits), bias ? bias->data_ptr<float>() : nullptr,
                   ids.data_ptr<int>(), weights.data_ptr<float>(), (int)T,
                   (int)E, (int)k, score == 1, (int)groups, (int)kept,
                   (int)best, renorm, (float)scale, cur_stream());
}

// A call's rows are taken so many at a time that each part of its workspace
// stays within 4 GiB and every offset into the rows within 32 bits.
constexpr int64_t kMoeRows = 1 << 17;

void moe_mlp(const torch::Tensor& X, const torch::Tensor& ids,
             const torch::Tensor& weights, const torch::Tensor& W1,
             const torch::Tensor* S1, const c10::optional<torch::Tensor>& b1,
             const torch::Tensor& W2, const torch::Tensor* S2,
             const c10::optional<torch::Tensor>& b2, const torch::Tensor& Y,
             const c10::optional<torch::Tensor>& residual, int64_t act) {
  const bool fp8 = S1 != nullptr;
  check_type(X, torch::kBFloat16, "X");
  check_rows(X, "X");
  const int64_t T = X.size(0), D = X.size(1);
  TORCH_CHECK(ids.dim() == 2, "ids must be 2D");
  const int64_t k = ids.size(1);
  TORCH_CHECK(k >= 1 && k <= 64, "1 to 64 experts a row, got ", k);
  check_whole(ids, torch::kInt32, {T, k}, "ids");
  check_whole(weights, torch::kFloat32, {T, k}, "weights");
  TORCH_CHECK(W1.dim() == 3, "W1 must be 3D");
  const int64_t E = W1.size(0), H = W1.size(1);
  TORCH_CHECK(E >= 1 && E <= 1024, "1 to 1024 experts, got ", E);
  TORCH_CHECK(T < 1 << 30, "too many rows: ", T);
  TORCH_CHECK(D >= 1 && D <= 1 << 18 && H >= 1 && H <= 1 << 18,
              "widths must be 1 to 2^18, got ", D, " and ", H);
  const int64_t unit = fp8 ? 128 : 64;
  const int64_t Dp = (D + unit - 1) / unit * unit;
  const int64_t Hp = (H + unit - 1) / unit * unit;
  const auto wtype = fp8 ? kFp8 : torch::kBFloat16;
  check_whole(W1, wtype, {E, H, Dp}, "W1");
  check_whole(W2, wtype, {E, D, Hp}, "W2");
  check_aligned(W1, "W1");
  check_aligned(W2, "W2");
  check_type(Y, torch::kBFloat16, "Y");
  check_shape(Y, {T, D}, "Y");
  check_rows(Y, "Y");
  check_act(act);
  std::vector<std::pair<const torch::Tensor*, const char*>> all = {
      {&X, "X"}, {&ids, "ids"}, {&weights, "weights"},
      {&W1, "W1"}, {&W2, "W2"}, {&Y, "Y"}};
  if (fp8) {
    check_whole(*S1, torch::kFloat32, {E, blocks128(H), Dp / 128}, "S1");
    check_whole(*S2, torch::kFloat32, {E, blocks128(D), Hp / 128}, "S2");
    all.push_back({S1, "S1"});
    all.push_back({S2, "S2"});
  }
  if (b1) {
    check_whole(*b1, torch::kFloat32, {E, H}, "b1");
    all.push_back({&*b1, "b1"});
  }
  if (b2) {
    check_whole(*b2, torch::kFloat32, {E, D}, "b2");
    all.push_back({&*b2, "b2"});
  }
  if (residual) {
    check_type(*residual, torch::kBFloat16, "residual");
    check_shape(*residual, {T, D}, "residual");
    check_rows(*residual, "residual");
    all.push_back({&*residual, "residual"});
  }
  for (auto& [t, name] : all)
    if (t != &Y && !((t == &X || (residual && t == &*residual)) &&
                     same_place(Y, *t)))
      check_apart({{&Y, "Y"}, {t, name}});
  check_devices(all);
  if (T == 0) return;
  const c10::DeviceGuard guard(X.device());
  const int64_t chunk = std::min(
      {T, std::max<int64_t>(
              1, std::min(kMoeRows, (int64_t(1) << 31) / std::max(Dp, Hp)) / k),
       (int64_t(1) << 30) / Dp});
  MoeMlp m{};
  m.W1 = W1.data_ptr();
  m.W2 = W2.data_ptr();
  if (fp8) {
    m.S1 = S1->data_ptr<float>();
    m.S2 = S2->data_ptr<float>();
  }
  if (b1) m.b1 = b1->data_ptr<float>();
  if (b2) m.b2 = b2->data_ptr<float>();
  m.ldx = row_stride(X);
  m.ldy = row_stride(Y);
  m.ldr = residual ? row_stride(*residual) : 0;
  m.E = (int)E;
  m.k = (int)k;
  m.D = (int)D;
  m.H = (int)H;
  m.act = (int)act;
  m.fp8 = fp8;
  auto rows = [&](int64_t t) {
    m.X = (const char*)X.data_ptr() + t * m.ldx * 2;
    m.Y = (char*)Y.data_ptr() + t * m.ldy * 2;
    m.residual = residual
                     ? (const char*)residual->data_ptr() + t * m.ldr * 2
                     : nullptr;
    m.ids = ids.data_ptr<int>() + t * k;
    m.weights = weights.data_ptr<float>() + t * k;
    m.T = (int)std::min(chunk, T - t);
  };
  int64_t bytes = 0;
  for (int64_t t = 0; t < T; t += chunk) {
    rows(t);
    bytes = std::max(bytes, moe_mlp_workspace(m));
  }
  auto ws = torch::empty({bytes}, X.options().dtype(torch::kUInt8));
  for (int64_t t = 0; t < T; t += chunk) {
    rows(t);
    launch_moe_mlp(m, ws.data_ptr(), cur_stream());
  }
}

// Y[t] = residual[t] + sum_j weights[t,j] (act(X[t] @ W1[e]^T + b1[e])
//        @ W2[e]^T + b2[e]),  e = ids[t,j]; an id outside of 0..E-1 adds
// nothing. X, Y, residual bf16 [T,D]; W1 [E,H,D up to 64s], W2
// [E,D,H up to 64s] bf16, filled up with zeros. The activated rows are rounded
// to bf16, which the second product takes; where assignments are more than 16
// to 32, the weighted terms to f16 over a power of two for each 64 columns. All
// sums are f32.
void moe_mlp_bf16(torch::Tensor X, torch::Tensor ids, torch::Tensor weights,
                  torch::Tensor W1, c10::optional<torch::Tensor> b1,
                  torch::Tensor W2, c10::optional<torch::Tensor> b2,
                  torch::Tensor Y, c10::optional<torch::Tensor> residual,
                  int64_t act) {
  moe_mlp(X, ids, weights, W1, nullptr, b1, W2, nullptr, b2, Y, residual, act);
}

// the same on e4m3 weights, each expert's as quant_fp8 leaves them with
// block_rows 128. X and the activated rows are rounded to e4m3 with a scale for
// each 128 values, the terms as above.
void moe_mlp_fp8(torch::Tensor X, torch::Tensor ids, torch::Tensor weights,
                 torch::Tensor W1, torch::Tensor S1,
                 c10::optional<torch::Tensor> b1, torch::Tensor W2,
                 torch::Tensor S2, c10::optional<torch::Tensor> b2,
                 torch::Tensor Y, c10::optional<torch::Tensor> residual,
                 int64_t act) {
  moe_mlp(X, ids, weights, W1, &S1, b1, W2, &S2, b2, Y, residual, act);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("gemm_bf16", &gemm_bf16, "bf16 MFMA GEMM (A @ B^T + bias, act)");
  m.def("conv2d_bf16", &conv2d_bf16, "bf16 implicit-GEMM conv2d NHWC");
  m.def("maxpool_bf16", &maxpool_bf16);
  m.def("avgpool_bf16", &avgpool_bf16);
  m.def("global_mean_bf16", &global_mean_bf16);
  m.def("softmax_bf16", &softmax_bf16);
  m.def("softmax_bf16_out", &softmax_bf16_out);
  m.def("cast_f32_bf16", &cast_f32_bf16);
  m.def("cast_bf16_f32", &cast_bf16_f32);
  m.def("channel_pad_bf16", &channel_pad_bf16);
  m.def("cast_f32_pad_bf16", &cast_f32_pad_bf16);
  m.def("add_relu_bf16", &add_relu_bf16);
  m.def("bias_act_bf16", &bias_act_bf16);
  m.def("scale_shift_bf16", &scale_shift_bf16);
  m.def("layernorm_bf16", &layernorm_bf16);
  m.def("gemm_batched_bf16", &gemm_batched_bf16);
  m.def("gemm_strided_bf16", &gemm_strided_bf16);
  m.def("attn_fused_bf16", &attn_fused_bf16);
  m.def("quant_fp8", &quant_fp8, py::arg("X"), py::arg("Q"), py::arg("S"),
        py::arg("block_rows") = 1,
        "round to e4m3 with a scale for each block of 128 along K");
  m.def("gemm_fp8", &gemm_fp8, py::arg("A"), py::arg("SA"), py::arg("B"),
        py::arg("SB"), py::arg("C"), py::arg("bias") = py::none(),
        py::arg("residual") = py::none(), py::arg("act") = 0,
        "block-scaled fp8 MFMA GEMM: act(A @ B^T + bias + residual)");
  m.def("moe_logits", &moe_logits, py::arg("X"), py::arg("W"),
        py::arg("logits"), "router logits in f32");
  m.def("moe_route", &moe_route, py::arg("logits"), py::arg("bias"),
        py::arg("ids"), py::arg("weights"), py::arg("score") = 0,
        py::arg("groups") = 1, py::arg("kept") = 1, py::arg("best") = 1,
        py::arg("renorm") = true, py::arg("scale") = 1.0,
        "the experts of each row and their weights");
  m.def("moe_mlp_bf16", &moe_mlp_bf16, py::arg("X"), py::arg("ids"),
        py::arg("weights"), py::arg("W1"), py::arg("b1"), py::arg("W2"),
        py::arg("b2"), py::arg("Y"), py::arg("residual") = py::none(),
        py::arg("act") = 0, "weighted sum of each row's experts");
  m.def("moe_mlp_fp8", &moe_mlp_fp8, py::arg("X"), py::arg("ids"),
        py::arg("weights"), py::arg("W1"), py::arg("S1"), py::arg("b1"),
        py::arg("W2"), py::arg("S2"), py::arg("b2"), py::arg("Y"),
        py::arg("residual") = py::none(), py::arg("act") = 0,
        "weighted sum of each row's experts, on e4m3 weights");
  m.def("dwconv_bf16", [](torch::Tensor X, torch::Tensor W2,
                          c10::optional<torch::Tensor> bias,
                          c10::optional<torch::Tensor> residual,
                          torch::Tensor Y, int64_t R, int64_t S,
                          int64_t sh, int64_t sw, int64_t pt, int64_t pl,
                          int64_t act) {
    TORCH_CHECK(X.scalar_type() == torch::kBFloat16 && X.is_contiguous());
    TORCH_CHECK(Y.scalar_type() == torch::kBFloat16 && Y.is_contiguous());
    TORCH_CHECK(W2.scalar_type() == torch::kBFloat16 && W2.is_contiguous());
    const float* bptr = nullptr;
    if (bias) {
      TORCH_CHECK(bias->scalar_type() == torch::kFloat32);
      bptr = bias->data_ptr<float>();
    }
    const void* rptr = nullptr;
    if (residual) {
      TORCH_CHECK(residual->scalar_type() == torch::kBFloat16 &&
                  residual->is_contiguous());
      rptr = residual->data_ptr();
    }
    int N = X.size(0), H = X.size(1), Wd = X.size(2), C = X.size(3);
    int HO = Y.size(1), WO = Y.size(2);
    TORCH_CHECK(Y.size(3) == C && Y.size(0) == N);
    launch_dwconv_bf16(X.data_ptr(), W2.data_ptr(), bptr, rptr,
                       Y.data_ptr(), N, H, Wd, C, HO, WO, (int)R, (int)S,
                       (int)sh, (int)sw, (int)pt, (int)pl, (int)act,
                       c10::hip::getCurrentHIPStream());
  });
  m.def("gemm8p_bf16", [](torch::Tensor A, torch::Tensor B,
                          torch::Tensor C,
                          c10::optional<torch::Tensor> bias,
                          c10::optional<torch::Tensor> residual,
                          int64_t K, int64_t act) {
    check_bf16(A, "A");
    check_bf16(B, "B");
    int ldc = check_out2d(C, "C");
    int64_t M = C.size(0), N = C.size(1), Kp = B.size(1);
    const float* bptr = nullptr;
    if (bias) bptr = bias->data_ptr<float>();
    const void* rptr = nullptr;
    if (residual) rptr = residual->data_ptr();
    launch_gemm_8p(A.data_ptr(), B.data_ptr(), C.data_ptr(), bptr, rptr,
                   (int)M, (int)N, (int)K, (int)Kp, (int)act, ldc,
                   c10::hip::getCurrentHIPStream());
  });
  m.def("jpeg_decode_slots", [](torch::Tensor arena, torch::Tensor planes,
                                torch::Tensor flags, int64_t n,
                                int64_t slot_bytes) {
    TORCH_CHECK(arena.scalar_type() == torch::kUInt8 &&
                arena.is_contiguous() && arena.is_cuda());
    TORCH_CHECK(planes.scalar_type() == torch::kUInt8 &&
                planes.is_cuda() &&
                planes.numel() >= n * slot_bytes);
    TORCH_CHECK(flags.scalar_type() == torch::kUInt8 && flags.is_cuda() &&
                flags.numel() >= n);
    launch_jpeg_decode(arena.data_ptr(), planes.data_ptr(),
                       flags.data_ptr(), (int)n, slot_bytes,
                       c10::hip::getCurrentHIPStream());
  });
  m.def("resize_norm", &resize_norm);
  m.def("resize_norm_batch", &resize_norm_batch);
  // Pin an externally-allocated host buffer (e.g. a /dev/shm mapping the
  // decode workers write into) so H2D from it is a true async DMA.
  m.def("host_register", [](int64_t ptr, int64_t bytes) {
    hipError_t e = hipHostRegister(reinterpret_cast<void*>(ptr),
                                   (size_t)bytes, hipHostRegisterDefault);
    // a refusal is the answer, not an error for the next call to report
    if (e != hipSuccess) (void)hipGetLastError();
    return e == hipSuccess;
  });
  m.def("host_unregister", [](int64_t ptr) {
    (void)hipHostUnregister(reinterpret_cast<void*>(ptr));
  });
}

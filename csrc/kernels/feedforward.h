// Launch API of the feed-forward, 8-bit and distillation operators (pure C++,
// as kernels.h).  Pitches count elements.  Every launcher checks what its
// kernels assume and throws mcc::Error; none synchronises or allocates.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace mcc {
namespace gpu {

// whether a grid of x by y workgroups can be launched: fewer than 2^32 threads
// along x
inline bool launchable(int64_t x, int threads, int64_t y = 1) {
  return x * threads < ((int64_t)1 << 32) && y <= 65535;
}

// activations of a gated block (0..2 as ActKind)
enum GateAct : int { GATE_NONE = 0, GATE_RELU = 1, GATE_TANH = 2, GATE_SILU = 3, GATE_GELU = 4 };

// H = f(X Wg^T) * (X Wu^T), bf16.  X [M][ldx], Wg / Wu [F][ldw], H / G / U
// [M][F] contiguous; ldx, ldw multiples of 8, X, Wg, Wu 16-byte aligned, and
// columns D .. round_up(D, 8) of their rows readable and zero, unless `any`.  gate / up
// (both or neither): the two projections, kept for the backward pass.
struct GatedParams {
  int M = 0, D = 0, F = 0, act = GATE_SILU;
  const void* x = nullptr;
  const void* wg = nullptr;
  const void* wu = nullptr;
  int64_t ldx = 0, ldw = 0;
  void* h = nullptr;
  void* gate = nullptr;
  void* up = nullptr;
  bool any = false;  // up to kAnyRows rows of X: rows of any pitch, length and 2-byte alignment
  void* work = nullptr;  // gated_forward_bytes(M, D, F) bytes (0: none needed), 16-byte aligned
};
int64_t gated_forward_bytes(int M, int D, int F);
constexpr int kAnyRows = 32;
// Products of more than kSplitRows rows of X with up to kSplitOutputs outputs and rows
// of kSplitBytes and more may be split over K (gated_forward_bytes, linear_i8_bytes),
// others never are.
constexpr int kSplitRows = 16, kSplitBytes = 4096, kSplitOutputs = 1 << 20;
void gated_forward(const GatedParams& p, hipStream_t s);

// The backward pass of H = f(G) * U from dH [M][F] and the saved G, U [M][F]
// (all three contiguous bf16):
//
//   dG = dH * U * f'(G), dU = dH * f(G)      rounded to bf16
//   dX = dG Wg + dU Wu        bf16 [M][D] contiguous
//   dW = [dG | dU]^T X        bf16 [2 F][D] contiguous: dWg, then dWu
//
// X [M][ldx], Wg / Wu [F][ldw] as in the forward pass, but any pitch and any
// 2-byte alignment.  `work`: gated_backward_bytes(M, D, F) bytes, 256-byte
// aligned, nothing of it kept from call to call.
struct GatedBwdParams {
  int M = 0, D = 0, F = 0, act = GATE_SILU;
  const void* dh = nullptr;
  const void* gate = nullptr;
  const void* up = nullptr;
  const void* x = nullptr;
  const void* wg = nullptr;
  const void* wu = nullptr;
  int64_t ldx = 0, ldw = 0;
  void* dx = nullptr;
  void* dw = nullptr;
  void* work = nullptr;
};
int64_t gated_backward_bytes(int M, int D, int F);
void gated_backward(const GatedBwdParams& p, hipStream_t s);

// Y = f((Xq Wq^T) * sx[m] * sw[n] + b[n]); Xq [M][ldx], Wq [N][ldw] int8 with
// pitches and addresses of multiples of 16 and columns K .. round_up(K, 16)
// zero, Y [M][N] contiguous, bf16 or fp32.
struct LinearI8Params {
  int M = 0, N = 0, K = 0, act = 0;  // ActKind
  const void* x = nullptr;
  const void* w = nullptr;
  int64_t ldx = 0, ldw = 0;
  const float* sx = nullptr;
  const float* sw = nullptr;
  const float* bias = nullptr;  // optional
  void* y = nullptr;
  bool f32 = false;
  bool any = false;  // up to kAnyRows rows of X: rows of any pitch, length and alignment
  void* work = nullptr;  // linear_i8_bytes(M, N, K) bytes (0: none needed), 16-byte aligned
};
int64_t linear_i8_bytes(int M, int N, int K);
// the largest K whose sum of products of two int8 cannot pass 32 bits:
// 131071 * 128 * 128 < 2^31
constexpr int kLinearI8MaxK = 131071;
void linear_i8(const LinearI8Params& p, hipStream_t s);

// RMS norm with the residual's addition and an 8-bit output:
//
//   S = X + R (R optional);  Y = S * W / sqrt(mean(S^2) + eps)
//   scale[m] = max |Y[m]| / 127;  Q = rint(Y / scale), to even
//
// X, R [M][D] with pitches ldx, ldr, W [D], all bf16 or all fp32; sum [M][D]
// contiguous in their type (written when R is given), Q int8 [M][D]
// contiguous.  A row of zeros has scale 0; a row with a value that is not
// finite, or whose sum of squares is not (or is 0 with eps = 0 where values are
// not), has scale NaN and zeros in Q.
struct RmsnormI8Params {
  int M = 0, D = 0;
  bool f32 = false;
  const void* x = nullptr;
  const void* r = nullptr;
  int64_t ldx = 0, ldr = 0;
  const void* w = nullptr;
  float eps = 0.f;
  void* sum = nullptr;
  int8_t* q = nullptr;
  float* scale = nullptr;
};
constexpr int kRmsnormI8MaxD = 32768;  // a row stays in the registers of one workgroup
void rmsnorm_i8(const RmsnormI8Params& p, hipStream_t s);

// Distillation from a teacher's top logits.  Row m: student logits z [N] (pitch
// ldz, bf16 or fp32), teacher logits t [K] (bf16 or fp32) of the classes idx
// [K] (int32 or int64), both contiguous [M][K].  An entry is there when its
// class is in [0, N) and its logit is not -inf; with q = softmax(t / T) over
// the row's entries and p = softmax(z / T) over all classes
//
//   loss[m] = T^2 sum_k q_k (log q_k - log p_{idx_k})
//   dz[m][j] = scale * T * (p_j - sum_{k: idx_k = j} q_k)
//
// A row without entries has loss 0 and gradient 0.  dz [M][N] contiguous, fp32
// or in the logits' type; nullptr: the loss alone.  `work`:
// distill_bytes(M, N, logits in fp32) bytes (0: none needed).
struct DistillParams {
  int M = 0, N = 0, K = 0;
  const void* z = nullptr;
  int64_t ldz = 0;
  bool z_f32 = false;
  const void* t = nullptr;
  bool t_f32 = false;
  const void* idx = nullptr;
  bool idx64 = false;
  float temperature = 1.f, scale = 1.f;
  void* dz = nullptr;
  bool dz_f32 = false;
  float* loss = nullptr;
  void* work = nullptr;
};
constexpr int kDistillMaxK = 1024;
int64_t distill_bytes(int M, int N, bool z_f32);
void distill_kl(const DistillParams& p, hipStream_t s);

// Up to three matrices copied into rows of ldd bytes (a multiple of 16), zeros
// behind the cols bytes that exist; sources of any pitch and alignment.
struct PadRows {
  struct Matrix {
    const void* src = nullptr;
    void* dst = nullptr;
    int64_t ld = 0, ldd = 0, rows = 0, cols = 0;
    int64_t pieces = 0;  // rows * ldd / 16; 0: no matrix
  };
  Matrix m[3];
};
void pad_rows(const PadRows& p, hipStream_t s);

}  // namespace gpu
}  // namespace mcc

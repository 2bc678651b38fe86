// Launch API of the feed-forward, 8-bit and distillation operators (pure C++,
// as kernels.h).  Pitches count elements.  Every launcher checks what its
// kernels assume and throws mcc::Error; none synchronises or allocates.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace mcc {
namespace gpu {

// activations of a gated block (0..2 as ActKind)
enum GateAct : int { GATE_NONE = 0, GATE_RELU = 1, GATE_TANH = 2, GATE_SILU = 3, GATE_GELU = 4 };

// H = f(X Wg^T) * (X Wu^T), bf16.  X [M][ldx], Wg / Wu [F][ldw], H / G / U
// [M][F] contiguous; ldx, ldw multiples of 8, X, Wg, Wu 16-byte aligned, and
// columns D .. round_up(D, 8) of their rows readable and zero.  gate / up
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
};
void gated_forward(const GatedParams& p, hipStream_t s);

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
};
// the largest K whose sum of products of two int8 cannot pass 32 bits:
// 131071 * 128 * 128 < 2^31
constexpr int kLinearI8MaxK = 131071;
void linear_i8(const LinearI8Params& p, hipStream_t s);

}  // namespace gpu
}  // namespace mcc

// Copies of matrices into rows of whole 16-byte pieces, zeros behind the last
// column (feedforward.h: PadRows), for kernels that read their operands in such
// pieces.  One launch for all operands of a call; bytes, so that bf16 and 8-bit
// integers share it.  A piece that does not start on 16 bytes is cut out of the
// two aligned ones that hold it, where both lie inside the matrix; a copy runs
// at about the rate of memory for any pitch and alignment.
#include "feedforward.h"
#include "mcc/common.h"
#include "mfma.h"

namespace mcc {
namespace gpu {

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u8v __attribute__((ext_vector_type(8)));

// bytes c .. c+15 of row r, zeros past its end
__device__ __forceinline__ u4 piece(const PadRows::Matrix& m, int64_t r, int64_t c) {
  const char* p = static_cast<const char*>(m.src);
  const int64_t at = r * m.ld + c, size = (m.rows - 1) * m.ld + m.cols;
  const int off = (int)(reinterpret_cast<uintptr_t>(p + at) & 15);
  u4 v;
  if (off == 0 && at + 16 <= size) {
    v = *reinterpret_cast<const u4*>(p + at);
  } else if (off && at >= off && at - off + 32 <= size) {
    const u4 lo = *reinterpret_cast<const u4*>(p + at - off), hi = *reinterpret_cast<const u4*>(p + at - off + 16);
    u8v w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    w = off & 8 ? __builtin_shufflevector(w, w, 2, 3, 4, 5, 6, 7, 7, 7) : w;
    w = off & 4 ? __builtin_shufflevector(w, w, 1, 2, 3, 4, 5, 6, 7, 7) : w;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], off & 3);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t b = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + 4 * i + k < m.cols) b |= (uint32_t)(uint8_t)p[at + 4 * i + k] << (8 * k);
      v[i] = b;
    }
  }
  const int64_t n = m.cols - c;  // bytes that exist
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t left = n - 4 * i;
    v[i] = left >= 4 ? v[i] : left <= 0 ? 0u : v[i] & (0xffffffffu >> (32 - 8 * (int)left));
  }
  return v;
}

__global__ void __launch_bounds__(256) pad_rows_kernel(PadRows p) {
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const PadRows::Matrix& m = p.m[k];
    if (i >= 0 && i < m.pieces) {
      const int64_t per = m.ldd / 16, r = i / per, c = (i - r * per) * 16;
      *reinterpret_cast<u4*>(static_cast<char*>(m.dst) + r * m.ldd + c) = piece(m, r, c);
    }
    i -= m.pieces;
  }
}

}  // namespace

void pad_rows(const PadRows& p, hipStream_t s) {
  int64_t n = 0;
  for (const auto& m : p.m) {
    MCC_CHECK(m.pieces == 0 || (m.rows > 0 && m.cols > 0 && m.ld >= 0 && m.ldd % 16 == 0 && m.ldd >= m.cols &&
                                m.pieces == m.rows * (m.ldd / 16) && reinterpret_cast<uintptr_t>(m.dst) % 16 == 0),
              "pad_rows: bad matrix");
    n += m.pieces;
  }
  if (n == 0) return;
  MCC_CHECK(n < ((int64_t)1 << 32) - 256, "pad_rows: too large");
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p);
  MCC_CHECK(hipGetLastError() == hipSuccess, "pad_rows: launch failed");
}

}  // namespace gpu
}  // namespace mcc

// The product C[a][b] = sum_k A[a][k] B[b][k] for few B rows (tokens) and a
// long A (weights), in the byte units of tile_gemm.h, on the 16 x 16 MFMAs:
// lane (r, g) = (lane & 15, lane >> 4) holds 16 bytes of row r, 64 bytes of K a
// fragment, and ends with A rows 4g .. 4g+3 of B row r.
//
// With up to 32 B rows every byte of A is used for at most 32 products, so the
// weights' stream from memory is what counts.  A workgroup owns 16 A rows (of
// each matrix when GATED) and its NW waves take the 128-byte blocks of K in
// turn: each wave goes straight from memory into MFMA fragments with U blocks
// (2U A loads of 1 KiB each) in flight, no LDS, no barrier in the loop; the
// waves' sums meet in LDS at the end, in wave order.  Eight waves (NW) from 4 KiB
// of K on: one token, int8 8192 x 4096 9.7 -> 7.4 us, bf16 2 x 8192 x 4096 27.8
// -> 25.5 us (5.3 TB/s); four below, where eight would have less than one round
// of U blocks (2 x 16000 x 1024 11.2 us, with eight 15.0).  Fragment columns past
// the last B row repeat it and are not stored.
#pragma once

#include "tile_gemm.h"

namespace mcc {
namespace gpu {
namespace tile {

// us per 128 bytes of K and 256 workgroups of 16 A rows (one matrix or two) and
// 16 or 32 B rows, measured; fewer than 256 take as long
inline float few_rows_us(bool two, int fb, int64_t n) {
  const float us = two ? (fb == 1 ? 0.17f : 0.235f) : (fb == 1 ? 0.145f : 0.19f);
  return us * (n < kCus ? 1.f : (float)n / kCus);
}

// NM: matrices on the A side (2: a gate and its projection)
template <class E, int FB, int U, int NW, int NM>
struct FewRows {
  typedef typename E::frag frag;
  typedef typename E::acc acc_t;
  static constexpr int kRows = 16 * FB;
  // [wave][matrix][b row][16 a rows], 4 bytes each
  static constexpr int kLds = NW * NM * kRows * 16 * 4;

  static __device__ __forceinline__ void run(const Operands& p, char* lds, int a0, int b0) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const char* pa[NM];
    const char* pb[FB];
#pragma unroll
    for (int h = 0; h < NM; ++h) pa[h] = p.a[h] + (int64_t)min(a0 + r16, p.arows - 1) * p.lda + g * 16;
#pragma unroll
    for (int j = 0; j < FB; ++j) pb[j] = p.b + (int64_t)min(b0 + 16 * j + r16, p.brows - 1) * p.ldb + g * 16;

    acc_t acc[NM][FB];
#pragma unroll
    for (int h = 0; h < NM; ++h)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[h][j][e] = 0;

    constexpr int kStep = 128;
    const int64_t nfull = p.kbytes / kStep;
    int64_t blk = wave;
    for (; blk + (int64_t)(U - 1) * NW < nfull; blk += (int64_t)U * NW) {
      frag xa[U][NM][2], xb[U][FB][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t o = (blk + u * NW) * kStep;
#pragma unroll
        for (int h = 0; h < NM; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) xa[u][h][k] = *reinterpret_cast<const frag*>(pa[h] + o + 64 * k);
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) xb[u][j][k] = *reinterpret_cast<const frag*>(pb[j] + o + 64 * k);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int h = 0; h < NM; ++h)
#pragma unroll
            for (int j = 0; j < FB; ++j) acc[h][j] = E::mul(xa[u][h][k], xb[u][j][k], acc[h][j]);
    }
    for (; blk * kStep < p.kbytes; blk += NW) {  // what is left: pieces behind the end of K are zero on both sides
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t o = blk * kStep + 64 * k;
        const bool in = o + g * 16 < p.kbytes;
        const frag z = __builtin_bit_cast(frag, i32x4{0, 0, 0, 0});
        frag xb[FB];
#pragma unroll
        for (int j = 0; j < FB; ++j) {
          xb[j] = *reinterpret_cast<const frag*>(pb[j] + (in ? o : -(int64_t)(g * 16)));
          if (!in) xb[j] = z;
        }
#pragma unroll
        for (int h = 0; h < NM; ++h) {
          frag xa = *reinterpret_cast<const frag*>(pa[h] + (in ? o : -(int64_t)(g * 16)));
          if (!in) xa = z;
#pragma unroll
          for (int j = 0; j < FB; ++j) acc[h][j] = E::mul(xa, xb[j], acc[h][j]);
        }
      }
    }

    // lane (r16, g) holds A rows 4g .. 4g+3 of B row 16 j + r16
#pragma unroll
    for (int h = 0; h < NM; ++h)
#pragma unroll
      for (int j = 0; j < FB; ++j)
        *reinterpret_cast<acc_t*>(lds + (((wave * NM + h) * kRows + 16 * j + r16) * 16 + 4 * g) * 4) = acc[h][j];
    __syncthreads();
  }

  // sum of matrix h's product at (b row, a row) after run()
  template <class T>
  static __device__ __forceinline__ T sum(const char* lds, int h, int b, int a) {
    T v = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const T*>(lds + (((w * NM + h) * kRows + b) * 16 + a) * 4);
    return v;
  }
};

}  // namespace tile
}  // namespace gpu
}  // namespace mcc

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

#include <algorithm>

#include "feedforward.h"
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

// Groups of 16 (1) or 32 (2) B rows, or tiles (0), which take `tiles` us: what the measured times say; up to 32 rows the weights' way from memory
// counts, which many workgroups that stream share best
// (in us: the time of what is taken)
inline int rows_way(bool two, int64_t a16, int brows, int64_t steps, float tiles, float& us) {
  const int64_t n1 = a16 * ((brows + 15) / 16), n2 = a16 * ((brows + 31) / 32);
  const float us1 = few_rows_us(two, 1, n1) * (float)steps, us2 = few_rows_us(two, 2, n2) * (float)steps;
  us = brows <= 16 ? us1 : std::min(us1, us2);
  if (brows <= 16) return 1;
  if (brows > 32 && (tiles <= us || brows > 16 * 65535)) {
    us = tiles;
    return 0;
  }
  return us1 <= us2 ? 1 : 2;
}

// Into how many sums over K a product of few tiles (`f`: the smallest) is split, 1:
// not at all.  `other`: us of the best way without; `bytes`: of an output's partial
// sum; `weights`: bytes of A, which the step times, taken with operands in the caches,
// do not hold.  Joining is a launch with its pauses and 2 `bytes` a value of each sum.
// bf16 152 x 7248 x 1024 with G and U kept, 48 tiles: 41.9 us, in 5 sums 18.7.
inline int splits_of(const Form& f, int64_t arows, int64_t brows, int64_t steps, int bytes, int64_t weights,
                     float other) {
  const int64_t n = workgroups(f, arows, brows);
  int best = 1;
  if (brows <= kSplitRows) return best;  // (the waves of few_rows.h split K themselves: 4 x 4288 x 448 11.2 us, in sums 15.2)
  if (steps * 128 <= kSplitBytes + 128) return best;  // (nothing to gain on a launch; + 128: whatever the rounding of K)
  for (int S = 2; S <= 16 && n * S <= 2 * kCus && steps / S >= 4; ++S) {
    const float us = std::max(form_us(f, n * S, (steps + S - 1) / S), (float)weights / 5e6f) + 7.f +
                     (float)(S * arows * brows * 2 * bytes) / 4e6f;
    if (us < other) {
      other = us;
      best = S;
    }
  }
  return best;
}

// 16 bytes from any address: the two aligned pieces that hold them (each holds a
// byte that is wanted, so neither can lie in another page), cut together when
// all loads are on their way
struct Cut {
  uint32_t lo __attribute__((ext_vector_type(4))), hi __attribute__((ext_vector_type(4)));
  __device__ __forceinline__ void load(const char* p, int n) {  // the first n of them, n > 0
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    lo = *reinterpret_cast<const u4*>(a & ~(uintptr_t)15);
    hi = *reinterpret_cast<const u4*>((a + n - 1) & ~(uintptr_t)15);
  }
  __device__ __forceinline__ i32x4 get(int by) const {  // by = p % 16
    typedef uint32_t u8 __attribute__((ext_vector_type(8)));
    u8 w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    w = by & 8 ? __builtin_shufflevector(w, w, 2, 3, 4, 5, 6, 7, 7, 7) : w;
    w = by & 4 ? __builtin_shufflevector(w, w, 1, 2, 3, 4, 5, 6, 7, 7) : w;
    i32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (int)__builtin_amdgcn_alignbyte(w[i + 1], w[i], by & 3);
    return v;
  }
};
// bytes o .. o + 15 of a row of n, zeros behind its end
__device__ __forceinline__ i32x4 load_end(const char* row, int64_t o, int64_t n) {
  const int left = (int)min(n - o, (int64_t)16);
  i32x4 v = {0, 0, 0, 0};
  if (left <= 0) return v;
  Cut c;
  c.load(row + o, left);
  v = c.get((int)(reinterpret_cast<uintptr_t>(row + o) & 15));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = left - 4 * i;
    v[i] = b >= 4 ? v[i] : b <= 0 ? 0 : v[i] & (int)(0xffffffffu >> (32 - 8 * b));
  }
  return v;
}

// NM: matrices on the A side (2: a gate and its projection).  ANY: rows of any
// address, pitch and length instead of whole aligned pieces: the copy into padded
// rows would read the weights, write them and read them again (1 x 5500 x 12370
// int8 40 us, so 26; 32 x 4095 x 8192 gated 75, so 69).  Unaligned loads, which the
// hardware takes, took 35 and 101.
template <class E, int FB, int U, int NW, int NM, bool ANY = false>
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
    for (int h = 0; h < NM; ++h) pa[h] = p.a[h] + (int64_t)min(a0 + r16, p.arows - 1) * p.lda + (ANY ? 0 : g * 16);
#pragma unroll
    for (int j = 0; j < FB; ++j) pb[j] = p.b + (int64_t)min(b0 + 16 * j + r16, p.brows - 1) * p.ldb + (ANY ? 0 : g * 16);
    int ba[NM], bb[FB];  // of a row's pieces: where they start in an aligned one
    if constexpr (ANY) {
#pragma unroll
      for (int h = 0; h < NM; ++h) ba[h] = (int)(reinterpret_cast<uintptr_t>(pa[h]) & 15);
#pragma unroll
      for (int j = 0; j < FB; ++j) bb[j] = (int)(reinterpret_cast<uintptr_t>(pb[j]) & 15);
    }

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
      if constexpr (ANY) {
        Cut ca[U][NM][2], cb[U][FB][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t o = (blk + u * NW) * kStep + 16 * g;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int h = 0; h < NM; ++h) ca[u][h][k].load(pa[h] + o + 64 * k, 16);
#pragma unroll
            for (int j = 0; j < FB; ++j) cb[u][j][k].load(pb[j] + o + 64 * k, 16);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            frag xb[FB];
#pragma unroll
            for (int j = 0; j < FB; ++j) xb[j] = __builtin_bit_cast(frag, cb[u][j][k].get(bb[j]));
#pragma unroll
            for (int h = 0; h < NM; ++h) {
              const frag xa = __builtin_bit_cast(frag, ca[u][h][k].get(ba[h]));
#pragma unroll
              for (int j = 0; j < FB; ++j) acc[h][j] = E::mul(xa, xb[j], acc[h][j]);
            }
          }
        continue;
      }
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
        auto last = [&](const char* row) {
          if constexpr (ANY) return __builtin_bit_cast(frag, load_end(row, o + g * 16, p.kbytes));
          const frag v = *reinterpret_cast<const frag*>(row + (in ? o : -(int64_t)(g * 16)));
          return in ? v : z;
        };
        frag xb[FB];
#pragma unroll
        for (int j = 0; j < FB; ++j) xb[j] = last(pb[j]);
#pragma unroll
        for (int h = 0; h < NM; ++h) {
          const frag xa = last(pa[h]);
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

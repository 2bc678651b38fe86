// Backward pass of the gated feed-forward block (feedforward.h: GatedBwdParams).
//
//   1. gated_grad: dG, dU from dH, G, U, written twice: [M][2 Fp] for dX (whose
//      K runs along F) and transposed [2 F][Mp] for dW (whose K runs along M).
//   2. dX [M][D] = dGU [M][2 Fp] * WT [D][2 Fp]^T,  WT = both weights transposed
//   3. dW [2F][D] = dGUT [2F][Mp] * XT [D][Mp]^T
//
// Transposes instead of operands read across their rows: every product is then
// the one tile loop of tile_gemm.h, and the transposes move M D + 2 F D + 2 M F
// elements once more.  At 8192 x 4096 x 12288 that is 0.9 GB beside
// 3.3 TFLOP.  Up to 64 rows the weights' bytes are the whole cost: dX then reads
// the weights as they are (gated_dx_rows).
//
// dG and dU are rounded to bf16, the operand type of the matrix unit: an
// independent error of 2^-9 rms per term, so 2^-9 rms of the sum as well.
#include "feedforward.h"
#include "gate_act.h"
#include "kernels.h"
#include "mcc/common.h"
#include "tile_gemm.h"

#include <algorithm>

namespace mcc {
namespace gpu {

namespace {

using tile::Bf16;
using tile::Operands;
using tile::Tile;

constexpr int kTP = 64;             // transpose tile
constexpr int kTPitch = kTP + 2;    // LDS pitch: 33 dwords, so that 8 rows apart is 8 banks apart

__device__ __forceinline__ bf16x8 cvt8(const float (&v)[8]) {
  const bf16x4 a = cvt4(v[0], v[1], v[2], v[3]), b = cvt4(v[4], v[5], v[6], v[7]);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 8 elements from column c on of a row with n columns, zeros past its end.
// wide: the row starts on 16 bytes and n is a multiple of 8.
__device__ __forceinline__ bf16x8 get8(const bf16* row, int c, int n, bool wide) {
  if (wide) {
    if (c + 8 <= n) return load8(row + c);
  }
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = c + e < n ? row[c + e] : (bf16)0.f;
  return v;
}

// the 64 x 64 tile in LDS ([row][col]) to out[c0 + col][r0 + row], 8 rows a
// store: columns below cols, rows below rows_pad (a multiple of 8)
__device__ __forceinline__ void put_transposed(const bf16* t, bf16* out, int64_t ldo, int r0, int c0, int cols,
                                               int rows_pad) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 256 + threadIdx.x;
    const int p = i & 7, c = i >> 3;
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[(8 * p + e) * kTPitch + c];
    if (c0 + c < cols && r0 + 8 * p < rows_pad) store8(out + (int64_t)(c0 + c) * ldo + r0 + 8 * p, v);
  }
}

__device__ __forceinline__ void to_lds(bf16* t, int row, int c, const bf16x8& v) {
  // (pitch 33 dwords: 4-byte alignment)
  const uint32_t* s = reinterpret_cast<const uint32_t*>(&v);
  uint32_t* d = reinterpret_cast<uint32_t*>(t + row * kTPitch + c);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] = s[e];
}

// out[c][r] = in[r][c] for r < rows, zeros for r up to rows_pad
__global__ void __launch_bounds__(256) transpose_kernel(const bf16* in, int64_t ld, int rows, int cols, bool wide, bf16* out,
                                                        int64_t ldo, int rows_pad) {
  __shared__ bf16 t[kTP * kTPitch];
  const int c0 = blockIdx.x * kTP, r0 = blockIdx.y * kTP;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 256 + threadIdx.x;
    const int c = (i & 7) * 8, r = i >> 3;
    bf16x8 v = {};
    if (r0 + r < rows) v = get8(in + (int64_t)(r0 + r) * ld, c0 + c, cols, wide);
    to_lds(t, r, c, v);
  }
  __syncthreads();
  put_transposed(t, out, ldo, r0, c0, cols, rows_pad);
}

// dG, dU of a 64 x 64 tile: dgu[m][f], dgu[m][Fp + f] and dgut[f][m], dgut[F + f][m]
template <int ACT>
__global__ void __launch_bounds__(256) gated_grad_kernel(const bf16* dh, const bf16* gate, const bf16* up, int M, int F, int Fp,
                                                         int Mp, bool wide, bf16* dgu, bf16* dgut) {
  __shared__ bf16 tg[kTP * kTPitch], tu[kTP * kTPitch];
  const int f0 = blockIdx.x * kTP, m0 = blockIdx.y * kTP;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 256 + threadIdx.x;
    const int c = (i & 7) * 8, r = i >> 3, m = m0 + r, f = f0 + c;
    bf16x8 vg = {}, vu = {};
    if (m < M && f < F) {
      const int64_t at = (int64_t)m * F;
      const bf16x8 d8 = get8(dh + at, f, F, wide), g8 = get8(gate + at, f, F, wide), u8 = get8(up + at, f, F, wide);
      float a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float fv, dv;
        gate_slope<ACT>((float)g8[e], fv, dv);
        const float d = (float)d8[e];
        a[e] = d * (float)u8[e] * dv;
        b[e] = d * fv;
      }
      vg = cvt8(a);
      vu = cvt8(b);
    }
    if (m < M && f < Fp) {
      store8(dgu + (int64_t)m * 2 * Fp + f, vg);
      store8(dgu + (int64_t)m * 2 * Fp + Fp + f, vu);
    }
    to_lds(tg, r, c, vg);
    to_lds(tu, r, c, vu);
  }
  __syncthreads();
  put_transposed(tg, dgut, Mp, m0, f0, F, Mp);
  put_transposed(tu, dgut + (int64_t)F * Mp, Mp, m0, f0, F, Mp);
}

// C[b][a] of the tile loop, bf16, or one of gridDim.y partial sums over K in fp32
template <int FA, int FB, int KS, int NST, int WPE, class TO>
__global__ void __launch_bounds__(tile::kThreads, WPE) tile_store_kernel(Operands op, TO* out, int steps) {
  typedef Tile<Bf16, FA, FB, KS, NST, false> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int ta, tb;
  tile::tile_of(cdiv(op.arows, T::RA), cdiv(op.brows, T::RB), ta, tb);
  const int a0 = ta * T::RA, b0 = tb * T::RB;
  const int nk = (int)((op.kbytes + KS - 1) / KS);
  const int k0 = blockIdx.y * steps;
  T t;
  t.run(op, lds, a0, b0, k0, min(nk, k0 + steps));

  const int wave = threadIdx.x >> 6, wa = wave >> 1, wb = wave & 1;
  out += (int64_t)blockIdx.y * op.arows * op.brows;
  const bool wide = op.arows % 8 == 0;
  typedef tile::RowStore<TO, FA> Rows;
  const Rows rows{lds + wave * Rows::kBytes};
  static_assert(4 * Rows::kBytes <= T::kLds, "row buffers fit the images");
  __syncthreads();  // every wave has read the last image
#pragma unroll
  for (int j = 0; j < FB; ++j) {
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = t.acc[i][j][e];
      rows.put(i, v);
    }
    rows.flush(out, b0 + T::b_out(wb, j, 0), a0 + T::a_out(wa, 0, 0), op.brows, op.arows, wide);
  }
}

// out = the sum of S partial arrays of n, in order
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* part, int64_t n, int S, bf16* out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if (n % 4 == 0) {
    f32x4 a = *reinterpret_cast<const f32x4*>(part + i);
    for (int s = 1; s < S; ++s) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(part + s * n + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += b[e];
    }
    *reinterpret_cast<bf16x4*>(out + i) = cvt4(a[0], a[1], a[2], a[3]);
  } else {
    for (int64_t e = i; e < std::min<int64_t>(i + 4, n); ++e) {
      float a = part[e];
      for (int s = 1; s < S; ++s) a += part[s * n + e];
      out[e] = (bf16)a;
    }
  }
}

// outputs a workgroup, workgroups a CU, us a step (tile_gemm.h: Form)
constexpr tile::Form kForms[] = {{64, 64, 2, 0.22f, 0.5f}, {128, 64, 2, 0.33f, 0.67f}, {128, 128, 2, 0.46f, 0.97f},
                                 {256, 256, 1, 1.55f, 1.55f}};
// How a product is done: its form, and into how many sums over K it is split
// where it has few tiles (1024 x 777 outputs, K = 5472: 37.0 us in 56 tiles of
// 128 x 128, 15.5 in 4 sums of them and 5 to add these up; 21.8 in 208 tiles of
// 64 x 64)
struct How {
  int form, S;
};
How how_of(int64_t arows, int64_t brows, int64_t kbytes) {
  const int64_t steps = (kbytes + 127) / 128;
  How best{0, 1};
  float least = 1e30f;
  for (int f = 0; f < 4; ++f) {
    const int64_t n = tile::workgroups(kForms[f], arows, brows);
    // (the largest form has no split: it is for products that fill the chip)
    for (int S = 1; S <= (f == 3 ? 1 : 16) && steps / S >= 4; S *= 2) {
      const float join = S == 1 ? 0.f : 4.f + (float)S * arows * brows * 8.f / 4e6f;
      const float us = tile::step_us(kForms[f], n * S) * (float)((steps + S - 1) / S) + join;
      if (us < least) {
        least = us;
        best = {f, S};
      }
    }
    if (steps < 4 && tile::step_us(kForms[f], n) < least) {
      least = tile::step_us(kForms[f], n);
      best = {f, 1};
    }
  }
  return best;
}

struct Plan {
  int Fp, Mp;
  How x, w;  // dX and dW
  int64_t dgu, dgut, wt, xt, part, total;  // byte offsets
};
Plan plan_of(int M, int D, int F) {
  Plan q;
  q.Fp = (int)round_up(F, 8);
  q.Mp = (int)round_up(M, 8);
  q.x = how_of(D, M, 4 * (int64_t)q.Fp);
  q.w = how_of(D, 2 * (int64_t)F, 2 * (int64_t)q.Mp);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += round_up(bytes, 256);
    return o;
  };
  q.dgu = take(2 * (int64_t)M * 2 * q.Fp);
  q.dgut = take(2 * 2 * (int64_t)F * q.Mp);
  q.wt = take(2 * (int64_t)D * 2 * q.Fp);
  q.xt = take(2 * (int64_t)D * q.Mp);
  const int64_t px = q.x.S > 1 ? 4 * q.x.S * (int64_t)M * D : 0, pw = q.w.S > 1 ? 4 * q.w.S * 2 * (int64_t)F * D : 0;
  q.part = take(std::max(px, pw));
  q.total = at;
  return q;
}

template <int FA, int FB, int NST, int WPE, class TO>
void launch_tiles(const Operands& o, TO* out, int steps, int S, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv(o.arows, 64 * FA) * cdiv(o.brows, 64 * FB)), (unsigned)S);
  hipLaunchKernelGGL((tile_store_kernel<FA, FB, 128, NST, WPE, TO>), grid, dim3(tile::kThreads), 0, s, o, out, steps);
}
template <class TO> void launch_form(int form, const Operands& o, TO* out, int steps, int S, hipStream_t s) {
  if (form == 0) launch_tiles<1, 1, 4, 2, TO>(o, out, steps, S, s);
  else if (form == 1) launch_tiles<2, 1, 3, 2, TO>(o, out, steps, S, s);
  else launch_tiles<2, 2, 2, 2, TO>(o, out, steps, S, s);
}

// out [brows][arows] = B A^T
void product(const char* a, int arows, const char* b, int brows, int64_t kbytes, bf16* out, float* part, How how,
             hipStream_t s) {
  Operands o;
  o.a[0] = o.a[1] = a;
  o.b = b;
  o.lda = o.ldb = kbytes;
  o.arows = arows;
  o.brows = brows;
  o.kbytes = kbytes;
  MCC_CHECK(kbytes <= (1 << 23), "gated_linear_bwd: row too long");
  const int steps = (int)((kbytes + 127) / 128);
  const int per = cdiv(steps, how.S), S = cdiv(steps, per);
  if (how.form == 3) {
    launch_tiles<4, 4, 2, 1, bf16>(o, out, steps, 1, s);
  } else if (S == 1) {
    launch_form<bf16>(how.form, o, out, steps, 1, s);
  } else {
    launch_form<float>(how.form, o, part, per, S, s);
    const int64_t n = (int64_t)arows * brows;
    hipLaunchKernelGGL(sum_partials_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s, part, n, S, out);
  }
}

void transpose(const void* in, int64_t ld, int rows, int cols, bf16* out, int64_t ldo, int rows_pad, hipStream_t s) {
  const bool wide = reinterpret_cast<uintptr_t>(in) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0;
  hipLaunchKernelGGL(transpose_kernel, dim3((unsigned)cdiv(cols, kTP), (unsigned)cdiv(rows, kTP)), dim3(256), 0, s,
                     static_cast<const bf16*>(in), ld, rows, cols, wide, out, ldo, rows_pad);
}

}  // namespace

int64_t gated_backward_bytes(int M, int D, int F) { return plan_of(M, D, F).total; }

void gated_backward(const GatedBwdParams& p, hipStream_t s) {
  MCC_CHECK(p.M > 0 && p.D > 0 && p.F > 0, "gated_linear_bwd: empty problem");
  MCC_CHECK(p.act >= GATE_NONE && p.act <= GATE_GELU, "gated_linear_bwd: unknown activation");
  MCC_CHECK(p.ldx >= p.D && p.ldw >= p.D, "gated_linear_bwd: row pitch");
  MCC_CHECK(p.M <= 4000000 && p.F <= (1 << 20), "gated_linear_bwd: too many rows");
  MCC_CHECK(reinterpret_cast<uintptr_t>(p.work) % 256 == 0, "gated_linear_bwd: workspace alignment");
  const Plan q = plan_of(p.M, p.D, p.F);
  char* w = static_cast<char*>(p.work);
  bf16* dgu = reinterpret_cast<bf16*>(w + q.dgu);
  bf16* dgut = reinterpret_cast<bf16*>(w + q.dgut);
  bf16* wt = reinterpret_cast<bf16*>(w + q.wt);
  bf16* xt = reinterpret_cast<bf16*>(w + q.xt);
  float* part = reinterpret_cast<float*>(w + q.part);

  const bool wide = p.F % 8 == 0 && (reinterpret_cast<uintptr_t>(p.dh) | reinterpret_cast<uintptr_t>(p.gate) |
                                     reinterpret_cast<uintptr_t>(p.up)) % 16 == 0;
  const dim3 grid((unsigned)cdiv(p.F, kTP), (unsigned)cdiv(p.M, kTP));
  with_gate(p.act, [&](auto k) {
    hipLaunchKernelGGL((gated_grad_kernel<decltype(k)::v>), grid, dim3(256), 0, s, static_cast<const bf16*>(p.dh),
                       static_cast<const bf16*>(p.gate), static_cast<const bf16*>(p.up), p.M, p.F, q.Fp, q.Mp, wide, dgu,
                       dgut);
  });
  transpose(p.wg, p.ldw, p.F, p.D, wt, 2 * q.Fp, q.Fp, s);
  transpose(p.wu, p.ldw, p.F, p.D, wt + q.Fp, 2 * q.Fp, q.Fp, s);
  transpose(p.x, p.ldx, p.M, p.D, xt, q.Mp, q.Mp, s);
  product(reinterpret_cast<const char*>(wt), p.D, reinterpret_cast<const char*>(dgu), p.M, 4 * (int64_t)q.Fp,
          static_cast<bf16*>(p.dx), part, q.x, s);
  product(reinterpret_cast<const char*>(xt), p.D, reinterpret_cast<const char*>(dgut), 2 * p.F, 2 * (int64_t)q.Mp,
          static_cast<bf16*>(p.dw), part, q.w, s);
  MCC_CHECK(hipGetLastError() == hipSuccess, "gated_linear_bwd: launch failed");
}

}  // namespace gpu
}  // namespace mcc

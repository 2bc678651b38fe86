// Product of 8-bit integers with a scale per token and per output channel:
//
//   Y[m][n] = f((sum_k Xq[m][k] Wq[n][k]) * sx[m] * sw[n] + b[n])
//
// The sum is exact: 32-bit integer accumulators, K bounded so that no sum of
// products can pass them.  It becomes a 32-bit float (one rounding), is scaled
// by the product of the two scales (two roundings), biased, and rounded to the
// output's type.
//
// Bound like the bf16 block of gated.hip, at half the bytes and twice the rate: 1 x
// 8192 x 4096 7.4 us (34 MB at 4.5 TB/s, the launch with it), 640 x 1000 x 4096 10.0
// (operands' way to LDS, 78 KB per us and CU), 8192 x 12288 x 4096 327-355 (2.5 Pop/s).
#include "feedforward.h"
#include "few_rows.h"
#include "gate_act.h"
#include "kernels.h"
#include "mcc/common.h"
#include "tile_gemm.h"

namespace mcc {
namespace gpu {

namespace {

using tile::FewRows;
using tile::I8;
using tile::Operands;
using tile::Tile;

// ReLU that keeps a NaN (a row whose scale is NaN stays visible)
template <int A> __device__ __forceinline__ float act_i8(float v) {
  if constexpr (A == ACT_RELU) return v < 0.f ? 0.f : v;
  else if constexpr (A == ACT_TANH) return tanh_(v);
  else return v;
}

template <int FA, int FB, int KS, int NST, int WPE, int ACT, class TO>
__global__ void __launch_bounds__(tile::kThreads, WPE) i8_tile_kernel(LinearI8Params p, Operands op) {
  typedef Tile<I8, FA, FB, KS, NST, false> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int ta, tb;
  tile::tile_of((int)blockIdx.x, cdiv(p.N, T::RA), cdiv(p.M, T::RB), ta, tb);
  const int n0 = ta * T::RA, m0 = tb * T::RB;
  T t;
  t.run(op, lds, n0, m0, 0, (int)((op.kbytes + KS - 1) / KS));

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r32 = lane & 31, g = lane >> 5, wa = wave >> 1, wb = wave & 1;
  const bool wide = p.N % 8 == 0;
  typedef tile::RowStore<TO, FA, FA * FB >= 12> Rows;
  const Rows rows{lds + wave * Rows::kBytes};
  // the tile's scales and biases, one of each per thread, dealt out through LDS
  float* sw = reinterpret_cast<float*>(lds + 4 * Rows::kBytes);
  float* bias = sw + T::RA;
  float* sx = bias + T::RA;
  static_assert(T::RA <= tile::kThreads && T::RB <= tile::kThreads, "one value per thread");
  static_assert(4 * Rows::kBytes + 4 * (2 * T::RA + T::RB) <= T::kLds, "row buffers and scales fit the images");
  const int tid = threadIdx.x, n = min(n0 + tid, p.N - 1);
  const float swv = p.sw[n], bv = p.bias ? p.bias[n] : 0.f, sxv = p.sx[min(m0 + tid, p.M - 1)];
  __syncthreads();  // every wave has read the last image
  if (tid < T::RA) {
    sw[tid] = swv;
    bias[tid] = bv;
  }
  if (tid < T::RB) sx[tid] = sxv;
  __syncthreads();
  f32x4 ws[FA][4], wb4[FA][4];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ws[i][e] = *reinterpret_cast<const f32x4*>(sw + T::a_out(wa, i, g) + 4 * e);
      wb4[i][e] = *reinterpret_cast<const f32x4*>(bias + T::a_out(wa, i, g) + 4 * e);
    }
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const float xs = sx[T::b_out(wb, j, r32)];
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[e] = act_i8<ACT>((float)t.acc[i][j][e] * (xs * ws[i][e >> 2][e & 3]) + wb4[i][e >> 2][e & 3]);
      rows.put(i, v);
    }
    rows.flush(static_cast<TO*>(p.y), m0 + T::b_out(wb, j, 0), n0 + T::a_out(wa, 0, 0), p.M, p.N, wide);
  }
}

// One of gridDim.y splits of K: partial sums [split][M][N], 32-bit integers
template <int FA, int FB, int KS, int NST, int WPE>
__global__ void __launch_bounds__(tile::kThreads, WPE) i8_part_kernel(LinearI8Params p, Operands op, int steps) {
  typedef Tile<I8, FA, FB, KS, NST, false> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int ta, tb;
  tile::tile_of((int)blockIdx.x, cdiv(p.N, T::RA), cdiv(p.M, T::RB), ta, tb);
  const int n0 = ta * T::RA, m0 = tb * T::RB;
  const int nk = (int)((op.kbytes + KS - 1) / KS), k0 = (int)blockIdx.y * steps;
  T t;
  t.run(op, lds, n0, m0, k0, min(nk, k0 + steps));

  const int wave = threadIdx.x >> 6, wa = wave >> 1, wb = wave & 1;
  typedef tile::RowStore<float, FA> Rows;  // (of the integers' bits)
  const Rows rows{lds + wave * Rows::kBytes};
  static_assert(4 * Rows::kBytes <= T::kLds, "row buffers fit the images");
  __syncthreads();  // every wave has read the last image
  float* out = static_cast<float*>(p.work) + (int64_t)blockIdx.y * p.M * p.N;
#pragma unroll
  for (int j = 0; j < FB; ++j) {
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = __builtin_bit_cast(float, (int)t.acc[i][j][e]);
      rows.put(i, v);
    }
    rows.flush(out, m0 + T::b_out(wb, j, 0), n0 + T::a_out(wa, 0, 0), p.M, p.N, p.N % 4 == 0);
  }
}
template <class TO> __global__ void __launch_bounds__(256) i8_join_kernel(LinearI8Params p, int S) {
  const int64_t size = (int64_t)p.M * p.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size) return;
  const int* part = static_cast<const int*>(p.work) + i;
  int v = 0;
#pragma unroll 4
  for (int s = 0; s < S; ++s) v += part[s * size];
  const int m = (int)(i / p.N), n = (int)(i - (int64_t)m * p.N);
  const float b = p.bias ? p.bias[n] : 0.f;
  with_act(p.act, [&](auto k) {
    static_cast<TO*>(p.y)[i] = (TO)act_i8<decltype(k)::v>((float)v * (p.sx[m] * p.sw[n]) + b);
  });
}

template <int FB, int U, int NW, bool ANY, class TO>
__global__ void __launch_bounds__(64 * NW) i8_rows_kernel(LinearI8Params p, Operands op) {
  typedef FewRows<I8, FB, U, NW, 1, ANY> R;
  __shared__ __attribute__((aligned(16))) char lds[R::kLds];
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * R::kRows;
  R::run(op, lds, n0, m0);
  TO* y = static_cast<TO*>(p.y);
  with_act(p.act, [&](auto k) {
    for (int i = threadIdx.x; i < R::kRows * 16; i += 64 * NW) {
      const int n = n0 + (i & 15), m = m0 + (i >> 4);
      if (n >= p.N || m >= p.M) continue;
      const int v = R::template sum<int>(lds, 0, i >> 4, i & 15);
      const float b = p.bias ? p.bias[n] : 0.f;
      y[(int64_t)m * p.N + n] = (TO)act_i8<decltype(k)::v>((float)v * (p.sx[m] * p.sw[n]) + b);
    }
  });
}

template <int FA, int FB, int KS, int NST, int WPE, class TO>
void launch_tiles(const LinearI8Params& p, const Operands& o, hipStream_t s) {
  const int64_t n = (int64_t)cdiv(p.N, 64 * FA) * cdiv(p.M, 64 * FB);
  MCC_CHECK(launchable(n, tile::kThreads), "linear_i8: too many rows");
  const dim3 grid((unsigned)n);
  if (p.act == ACT_RELU)
    hipLaunchKernelGGL((i8_tile_kernel<FA, FB, KS, NST, WPE, ACT_RELU, TO>), grid, dim3(tile::kThreads), 0, s, p, o);
  else if (p.act == ACT_TANH)
    hipLaunchKernelGGL((i8_tile_kernel<FA, FB, KS, NST, WPE, ACT_TANH, TO>), grid, dim3(tile::kThreads), 0, s, p, o);
  else
    hipLaunchKernelGGL((i8_tile_kernel<FA, FB, KS, NST, WPE, ACT_NONE, TO>), grid, dim3(tile::kThreads), 0, s, p, o);
}

// outputs a workgroup, workgroups a CU, us a step and for the ends: 640 x 1000 x 4096
// 9.8 / 11.6 / 16.1 / - / 37.6 us, 2048^3 16.8 / 15.2 / 13.1 / - / 25.3, 1024 x 4096 x
// 4096 29.4 / 25.7 / 22.6 / - / 40.3, 4096^3 117 / 91 / 68 / - / 60 (and 256 x 128
// tiles, which win nowhere, 23.0, 17.7, 29.5, 69); the fourth is for sizes that leave
// a last round of the others half empty: 3596 x 3944 x 2752 73.9 us without it, 57.8
// with
constexpr tile::Form kForms[] = {{64, 64, 2, 0.21f, 0.45f, 0.6f}, {128, 64, 2, 0.28f, 0.69f, 0.8f},
                                 {128, 128, 2, 0.6f, 1.03f, 1.2f}, {256, 192, 1, 1.4f, 1.4f, 3.5f},
                                 {256, 256, 1, 1.75f, 1.75f, 4.f}};

struct Plan {
  int form, way, S;  // S > 1: the first form, split
};
Plan plan_of(int M, int N, int64_t kbytes, bool any) {
  const int64_t steps = (kbytes + 127) / 128;
  Plan q;
  q.form = tile::best_form(kForms, N, M, steps);
  const float tiles = tile::form_us(kForms[q.form], tile::workgroups(kForms[q.form], N, M), steps);
  float us;
  q.way = tile::rows_way(false, cdiv(N, 16), M, steps, tiles, us);
  q.S = any ? 1 : tile::splits_of(kForms[0], N, M, steps, 4, N * kbytes, us);
  return q;
}

template <class TO> void launch(const LinearI8Params& p, hipStream_t s) {
  Operands o;
  o.a[0] = o.a[1] = static_cast<const char*>(p.w);
  o.b = static_cast<const char*>(p.x);
  o.lda = p.ldw;
  o.ldb = p.ldx;
  o.arows = p.N;
  o.brows = p.M;
  o.kbytes = p.any ? p.K : round_up(p.K, 16);
  const Plan q = plan_of(p.M, p.N, o.kbytes, p.any);
  if (q.S > 1) {
    MCC_CHECK(p.work != nullptr && reinterpret_cast<uintptr_t>(p.work) % 16 == 0, "linear_i8: workspace missing");
    const int steps = (int)((o.kbytes + 127) / 128), per = cdiv(steps, q.S), S = cdiv(steps, per);
    const int64_t n = (int64_t)p.M * p.N;  // (at most two workgroups a CU of the first form: a small number)
    hipLaunchKernelGGL((i8_part_kernel<1, 1, 128, 4, 2>), dim3((unsigned)(cdiv(p.N, 64) * cdiv(p.M, 64)), (unsigned)S),
                       dim3(tile::kThreads), 0, s, p, o, per);
    hipLaunchKernelGGL(i8_join_kernel<TO>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, S);
  } else if (q.way == 1) {
    const dim3 grid((unsigned)cdiv(p.N, 16), (unsigned)cdiv(p.M, 16));
    const bool eight = o.kbytes >= 4096;
    MCC_CHECK(launchable(grid.x, eight ? 512 : 256, grid.y), "linear_i8: too many output columns");
    if (p.any && eight) hipLaunchKernelGGL((i8_rows_kernel<1, 2, 8, true, TO>), grid, dim3(512), 0, s, p, o);
    else if (p.any) hipLaunchKernelGGL((i8_rows_kernel<1, 2, 4, true, TO>), grid, dim3(256), 0, s, p, o);
    else if (eight) hipLaunchKernelGGL((i8_rows_kernel<1, 4, 8, false, TO>), grid, dim3(512), 0, s, p, o);
    else hipLaunchKernelGGL((i8_rows_kernel<1, 4, 4, false, TO>), grid, dim3(256), 0, s, p, o);
  } else if (q.way == 2) {
    const dim3 grid((unsigned)cdiv(p.N, 16), (unsigned)cdiv(p.M, 32));
    MCC_CHECK(launchable(grid.x, 256, grid.y), "linear_i8: too many output columns");
    if (p.any) hipLaunchKernelGGL((i8_rows_kernel<2, 2, 4, true, TO>), grid, dim3(256), 0, s, p, o);
    else hipLaunchKernelGGL((i8_rows_kernel<2, 2, 4, false, TO>), grid, dim3(256), 0, s, p, o);
  } else {
    switch (q.form) {
      case 0: launch_tiles<1, 1, 128, 4, 2, TO>(p, o, s); break;
      case 1: launch_tiles<2, 1, 128, 3, 2, TO>(p, o, s); break;
      case 2: launch_tiles<2, 2, 128, 2, 2, TO>(p, o, s); break;
      case 3: launch_tiles<4, 3, 128, 2, 1, TO>(p, o, s); break;
      default: launch_tiles<4, 4, 128, 2, 1, TO>(p, o, s); break;
    }
  }
  MCC_CHECK(hipGetLastError() == hipSuccess, "linear_i8: launch failed");
}

}  // namespace

int64_t linear_i8_bytes(int M, int N, int K) {
  const int S = plan_of(M, N, round_up(K, 16), false).S;
  return S > 1 ? (int64_t)S * M * N * 4 : 0;
}

void linear_i8(const LinearI8Params& p, hipStream_t s) {
  MCC_CHECK(p.M >= 0 && p.N > 0 && p.K > 0, "linear_i8: empty problem");
  MCC_CHECK(p.M <= (1 << 30) && p.N <= (1 << 30), "linear_i8: too many rows");
  MCC_CHECK(p.K <= kLinearI8MaxK, "linear_i8: K too large for an exact 32-bit sum");
  MCC_CHECK(p.act >= ACT_NONE && p.act <= ACT_TANH, "linear_i8: unknown activation");
  MCC_CHECK(!p.any || p.M <= kAnyRows, "linear_i8: too many rows of any alignment");
  MCC_CHECK(p.ldx >= 0 && p.ldw >= 0, "linear_i8: row pitch");
  MCC_CHECK(p.any || (p.ldx >= round_up(p.K, 16) && p.ldw >= round_up(p.K, 16) && p.ldx % 16 == 0 && p.ldw % 16 == 0),
            "linear_i8: row pitches must be multiples of 16");
  MCC_CHECK(p.any || (p.ldx < (1 << 23) && p.ldw < (1 << 23)), "linear_i8: row pitch too large");
  MCC_CHECK(p.any || (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) % 16 == 0,
            "linear_i8: operands must be 16-byte aligned");
  if (p.M == 0) return;
  if (p.f32) launch<float>(p, s);
  else launch<bf16>(p, s);
}

}  // namespace gpu
}  // namespace mcc

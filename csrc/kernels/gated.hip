// Gated feed-forward block, bf16:
//
//   G = X Wg^T, U = X Wu^T, H = f(G) * U          f: none, relu, tanh, silu, gelu
//
// Forward: one launch.  A tile multiplies the same X rows with the matching
// rows of both weights (tile_gemm.h, SPLIT), so a lane ends with G and U of the
// same outputs and the activation, the product and the rounding happen on the
// accumulators: H is rounded once from 32-bit sums, as are the G and U that a
// training step keeps.
//
// Bound by the weights' bytes for few rows (1 x 4096 x 8192 25.2 us, 134 MB at 5.3
// TB/s), by the operands' way to LDS between, about 73 to 91 KB per us and CU for small
// tiles (777 x 1024 x 2731 with G and U kept 21.5-22.5), by the matrix unit's power for many
// (8192 x 4096 x 12288 with G and U kept 1250, 1.32 PFLOP/s, of which the stores of
// 0.6 GB take 100; past the caches, as they no longer push out the operands).
#include "feedforward.h"
#include "few_rows.h"
#include "gate_act.h"
#include "kernels.h"
#include "mcc/common.h"
#include "tile_gemm.h"

namespace mcc {
namespace gpu {

namespace {

using tile::Bf16;
using tile::FewRows;
using tile::Operands;
using tile::Tile;

Operands operands(const GatedParams& p) {
  Operands o;
  o.a[0] = static_cast<const char*>(p.wg);
  o.a[1] = static_cast<const char*>(p.wu);
  o.b = static_cast<const char*>(p.x);
  o.lda = p.ldw * 2;
  o.ldb = p.ldx * 2;
  o.arows = p.F;
  o.brows = p.M;
  o.kbytes = (p.any ? p.D : round_up(p.D, 8)) * 2;
  return o;
}

template <int FA, int FB, int KS, int NST, int WPE, int ACT>
__global__ void __launch_bounds__(tile::kThreads, WPE) gated_tile_kernel(GatedParams p, Operands op) {
  typedef Tile<Bf16, FA, FB, KS, NST, true> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int ta, tb;
  tile::tile_of((int)blockIdx.x, cdiv(p.F, T::RA / 2), cdiv(p.M, T::RB), ta, tb);
  const int f0 = ta * (T::RA / 2), m0 = tb * T::RB;
  T t;
  t.run(op, lds, f0, m0, 0, (int)((op.kbytes + KS - 1) / KS));

  const int wave = threadIdx.x >> 6, wa = wave >> 1, wb = wave & 1;
  const bool wide = p.F % 8 == 0;
  typedef tile::RowStore<bf16, FA / 2, FA * FB >= 12> Rows;
  const Rows rows{lds + wave * Rows::kBytes};
  static_assert(4 * Rows::kBytes <= T::kLds, "row buffers fit the images");
  __syncthreads();  // every wave has read the last image
  const int f = f0 + T::a_out(wa, 0, 0);
  float v[16];
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const int m = m0 + T::b_out(wb, j, 0);
#pragma unroll
    for (int i = 0; i < FA / 2; ++i) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = gate_f<ACT>(t.acc[i][j][e]) * t.acc[FA / 2 + i][j][e];
      rows.put(i, v);
    }
    rows.flush(static_cast<bf16*>(p.h), m, f, p.M, p.F, wide);
    if (p.gate) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < FA / 2; ++i) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = t.acc[k * (FA / 2) + i][j][e];
          rows.put(i, v);
        }
        rows.flush(static_cast<bf16*>(k ? p.up : p.gate), m, f, p.M, p.F, wide);
      }
    }
  }
}

// The two projections of one of gridDim.y splits of K: partial sums [split][G | U][M][F]
template <int FA, int FB, int KS, int NST, int WPE>
__global__ void __launch_bounds__(tile::kThreads, WPE) gated_part_kernel(GatedParams p, Operands op, int steps) {
  typedef Tile<Bf16, FA, FB, KS, NST, true> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int ta, tb;
  tile::tile_of((int)blockIdx.x, cdiv(p.F, T::RA / 2), cdiv(p.M, T::RB), ta, tb);
  const int f0 = ta * (T::RA / 2), m0 = tb * T::RB;
  const int nk = (int)((op.kbytes + KS - 1) / KS), k0 = (int)blockIdx.y * steps;
  T t;
  t.run(op, lds, f0, m0, k0, min(nk, k0 + steps));

  const int wave = threadIdx.x >> 6, wa = wave >> 1, wb = wave & 1;
  typedef tile::RowStore<float, FA / 2> Rows;
  const Rows rows{lds + wave * Rows::kBytes};
  static_assert(4 * Rows::kBytes <= T::kLds, "row buffers fit the images");
  __syncthreads();  // every wave has read the last image
  float* out = static_cast<float*>(p.work) + (int64_t)blockIdx.y * 2 * p.M * p.F;
  float v[16];
#pragma unroll
  for (int j = 0; j < FB; ++j) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < FA / 2; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = t.acc[k * (FA / 2) + i][j][e];
        rows.put(i, v);
      }
      rows.flush(out + (int64_t)k * p.M * p.F, m0 + T::b_out(wb, j, 0), f0 + T::a_out(wa, 0, 0), p.M, p.F, p.F % 4 == 0);
    }
  }
}
__global__ void __launch_bounds__(256) gated_join_kernel(GatedParams p, int S) {
  const int64_t n = (int64_t)p.M * p.F, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float* part = static_cast<const float*>(p.work) + i;
  float g = 0.f, u = 0.f;
#pragma unroll 4
  for (int s = 0; s < S; ++s) {
    g += part[2 * s * n];
    u += part[(2 * s + 1) * n];
  }
  with_gate(p.act, [&](auto k) { static_cast<bf16*>(p.h)[i] = (bf16)(gate_f<decltype(k)::v>(g) * u); });
  if (p.gate) {
    static_cast<bf16*>(p.gate)[i] = (bf16)g;
    static_cast<bf16*>(p.up)[i] = (bf16)u;
  }
}

template <int FB, int U, int NW, bool ANY>
__global__ void __launch_bounds__(64 * NW) gated_rows_kernel(GatedParams p, Operands op) {
  typedef FewRows<Bf16, FB, U, NW, 2, ANY> R;
  __shared__ __attribute__((aligned(16))) char lds[R::kLds];
  const int f0 = blockIdx.x * 16, m0 = blockIdx.y * R::kRows;
  R::run(op, lds, f0, m0);
  bf16* h = static_cast<bf16*>(p.h);
  bf16* gate = static_cast<bf16*>(p.gate);
  bf16* up = static_cast<bf16*>(p.up);
  with_gate(p.act, [&](auto k) {
    for (int i = threadIdx.x; i < R::kRows * 16; i += 64 * NW) {
      const int f = f0 + (i & 15), m = m0 + (i >> 4);
      if (f >= p.F || m >= p.M) continue;
      const float gv = R::template sum<float>(lds, 0, i >> 4, i & 15);
      const float uv = R::template sum<float>(lds, 1, i >> 4, i & 15);
      const int64_t at = (int64_t)m * p.F + f;
      h[at] = (bf16)(gate_f<decltype(k)::v>(gv) * uv);
      if (gate) {
        gate[at] = (bf16)gv;
        up[at] = (bf16)uv;
      }
    }
  });
}

// outputs a workgroup (gate and projection at once), workgroups a CU, us a step and
// for the ends:
// 1024^3 256 workgroups of the first form 7.8 us, of the second (128) 10.3;
// 3000 x 512 x 4096 37.0 / 31.3 / 43.9 us; 1024 x 4096 x 4096 84 / 62 / 58 / - / 79;
// 4096^3 343 / 251 / 233 / - / 206; the fourth is for sizes that leave a last round
// of the others half empty: 2075 x 4248 x 11904 580 us without it, 435 with
constexpr tile::Form kForms[] = {{64, 64, 2, 0.27f, 0.67f, 1.6f}, {64, 128, 2, 0.46f, 0.97f, 3.7f},
                                 {128, 128, 1, 0.9f, 0.9f, 3.9f}, {128, 192, 1, 1.28f, 1.28f, 4.9f},
                                 {128, 256, 1, 1.61f, 1.61f, 5.9f}};

template <int FA, int FB, int NST, int WPE, int ACT>
void launch_tiles(const GatedParams& p, const Operands& o, hipStream_t s) {
  const int64_t n = (int64_t)cdiv(p.F, 32 * FA) * cdiv(p.M, 64 * FB);
  MCC_CHECK(launchable(n, tile::kThreads), "gated_linear: too many rows");
  const dim3 grid((unsigned)n);
  hipLaunchKernelGGL((gated_tile_kernel<FA, FB, 128, NST, WPE, ACT>), grid, dim3(tile::kThreads), 0, s, p, o);
}

struct Plan {
  int form, way, S;  // S > 1: the first form, split
};
Plan plan_of(int M, int F, int64_t kbytes, bool any) {
  const int64_t steps = (kbytes + 127) / 128;
  Plan q;
  q.form = tile::best_form(kForms, F, M, steps);
  const float tiles = tile::form_us(kForms[q.form], tile::workgroups(kForms[q.form], F, M), steps);
  float us;
  q.way = tile::rows_way(true, cdiv(F, 16), M, steps, tiles, us);
  q.S = any ? 1 : tile::splits_of(kForms[0], F, M, steps, 8, 2 * F * kbytes, us);
  return q;
}

}  // namespace

int64_t gated_forward_bytes(int M, int D, int F) {
  const int S = plan_of(M, F, round_up(D, 8) * 2, false).S;
  return S > 1 ? (int64_t)S * 2 * M * F * 4 : 0;
}

void gated_forward(const GatedParams& p, hipStream_t s) {
  MCC_CHECK(p.M >= 0 && p.D > 0 && p.F > 0, "gated_linear: empty problem");
  MCC_CHECK(p.M <= (1 << 30) && p.F <= (1 << 30), "gated_linear: too many rows");
  MCC_CHECK(p.act >= GATE_NONE && p.act <= GATE_GELU, "gated_linear: unknown activation");
  MCC_CHECK(!p.any || p.M <= kAnyRows, "gated_linear: too many rows of any alignment");
  MCC_CHECK(p.any || (p.ldx >= round_up(p.D, 8) && p.ldw >= round_up(p.D, 8) && p.ldx % 8 == 0 && p.ldw % 8 == 0),
            "gated_linear: row pitches must be multiples of 8");
  MCC_CHECK(p.any || (p.ldx < (1 << 22) && p.ldw < (1 << 22)), "gated_linear: row pitch too large");
  MCC_CHECK(p.ldx >= 0 && p.ldw >= 0, "gated_linear: row pitch");
  MCC_CHECK(p.any || (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.wg) | reinterpret_cast<uintptr_t>(p.wu)) %
                    16 == 0, "gated_linear: operands must be 16-byte aligned");
  MCC_CHECK((p.gate == nullptr) == (p.up == nullptr), "gated_linear: gate and up go together");
  if (p.M == 0) return;
  const Operands o = operands(p);
  const Plan q = plan_of(p.M, p.F, o.kbytes, p.any);
  if (q.S > 1) {
    MCC_CHECK(p.work != nullptr && reinterpret_cast<uintptr_t>(p.work) % 16 == 0, "gated_linear: workspace missing");
    const int steps = (int)((o.kbytes + 127) / 128), per = cdiv(steps, q.S), S = cdiv(steps, per);
    const int64_t n = (int64_t)p.M * p.F;  // (at most two workgroups a CU of the first form: a small number)
    hipLaunchKernelGGL((gated_part_kernel<2, 1, 128, 3, 2>), dim3((unsigned)(cdiv(p.F, 64) * cdiv(p.M, 64)), (unsigned)S),
                       dim3(tile::kThreads), 0, s, p, o, per);
    hipLaunchKernelGGL(gated_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, S);
  } else if (q.way == 1) {
    const dim3 grid((unsigned)cdiv(p.F, 16), (unsigned)cdiv(p.M, 16));
    const bool eight = o.kbytes >= 4096;
    MCC_CHECK(launchable(grid.x, eight ? 512 : 256, grid.y), "gated_linear: too many output columns");
    if (p.any && eight) hipLaunchKernelGGL((gated_rows_kernel<1, 2, 8, true>), grid, dim3(512), 0, s, p, o);
    else if (p.any) hipLaunchKernelGGL((gated_rows_kernel<1, 2, 4, true>), grid, dim3(256), 0, s, p, o);
    else if (eight) hipLaunchKernelGGL((gated_rows_kernel<1, 4, 8, false>), grid, dim3(512), 0, s, p, o);
    else hipLaunchKernelGGL((gated_rows_kernel<1, 4, 4, false>), grid, dim3(256), 0, s, p, o);
  } else if (q.way == 2) {
    const dim3 grid((unsigned)cdiv(p.F, 16), (unsigned)cdiv(p.M, 32));
    MCC_CHECK(launchable(grid.x, 256, grid.y), "gated_linear: too many output columns");
    if (p.any) hipLaunchKernelGGL((gated_rows_kernel<2, 2, 4, true>), grid, dim3(256), 0, s, p, o);
    else hipLaunchKernelGGL((gated_rows_kernel<2, 2, 4, false>), grid, dim3(256), 0, s, p, o);
  } else {
    with_gate(p.act, [&](auto k) {
      constexpr int A = decltype(k)::v;
      switch (q.form) {
        case 0: launch_tiles<2, 1, 3, 2, A>(p, o, s); break;
        case 1: launch_tiles<2, 2, 2, 2, A>(p, o, s); break;
        case 2: launch_tiles<4, 2, 3, 1, A>(p, o, s); break;
        case 3: launch_tiles<4, 3, 2, 1, A>(p, o, s); break;
        default: launch_tiles<4, 4, 2, 1, A>(p, o, s); break;
      }
    });
  }
  MCC_CHECK(hipGetLastError() == hipSuccess, "gated_linear: launch failed");
}

}  // namespace gpu
}  // namespace mcc

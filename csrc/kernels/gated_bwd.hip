// Backward pass of the gated feed-forward block (feedforward.h: GatedBwdParams).
//
//   1. gated_prepare: dG, dU from dH, G, U, written twice: [M][2 Fp] for dX
//      (whose K runs along F) and transposed [2 F][Mp] for dW (whose K runs
//      along M); X transposed, and the weights unless 2b. follows
//   2a. dX [M][D] = dGU [M][2 Fp] * WT [D][2 Fp]^T, or
//   2b. up to 128 rows dX from the weights as they are (gated_dx_rows_kernel)
//   3. dW [2F][D] = dGUT [2F][Mp] * XT [D][Mp]^T, in the launch of 2a. where that is
//      faster, with the sums of 2b. else
//   4. the sums of products that were split over K
//
// Transposes instead of operands read across their rows: every product is then
// the one tile loop of tile_gemm.h, and the transposes move M D + 2 F D + 2 M F
// elements once more.  At 8192 x 4096 x 12288 that is 0.9 GB (0.4 ms with dG and
// dU themselves) beside 3.3 TFLOP (2.35 ms, 1.4 PFLOP/s).  For few rows the weights' bytes are
// the whole cost, and 2b. reads them once.
//
// dG and dU are rounded to bf16, the operand type of the matrix unit: an
// independent error of at most 2^-8 per term, so no more of the sum's terms.
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

// A matrix to be read in runs of 8 columns from any 2-byte address and pitch.
struct Source {
  const bf16* p;
  int64_t ld, size;  // pitch, and elements from p to the last one
  int rows, cols;
};
Source source(const void* p, int64_t ld, int rows, int cols) {
  return Source{static_cast<const bf16*>(p), ld, (rows - 1) * ld + cols, rows, cols};
}
// columns c .. c+7 of row r, zeros where there are none.  A run that does not
// start on 16 bytes is cut out of the two aligned pieces that hold it, where
// both lie inside the matrix.
__device__ __forceinline__ bf16x8 get8(const Source& m, int r, int c) {
  bf16x8 v = {};
  if (r >= m.rows || c >= m.cols) return v;
  const int64_t at = r * m.ld + c;
  const uintptr_t a = reinterpret_cast<uintptr_t>(m.p + at);
  const int off = (int)(a & 15) / 2;
  if (off == 0 && at + 8 <= m.size) {
    v = load8(m.p + at);
  } else if (at - off >= 0 && at - off + 16 <= m.size) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u8 __attribute__((ext_vector_type(8)));
    const u4 lo = *reinterpret_cast<const u4*>(m.p + at - off), hi = *reinterpret_cast<const u4*>(m.p + at - off + 8);
    u8 w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    w = off & 4 ? __builtin_shufflevector(w, w, 2, 3, 4, 5, 6, 7, 7, 7) : w;
    w = off & 2 ? __builtin_shufflevector(w, w, 1, 2, 3, 4, 5, 6, 7, 7) : w;
    u4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], 2 * (off & 1));
    v = __builtin_bit_cast(bf16x8, o);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < m.cols ? m.p[at + e] : (bf16)0.f;
  }
#pragma unroll
  for (int e = 1; e < 8; ++e) v[e] = c + e < m.cols ? v[e] : (bf16)0.f;
  return v;
}

// the 64 x 64 tile in LDS ([row][col]) to out[c0 + col][r0 + row], 8 rows a
// store: columns below cols, rows below rows_pad (a multiple of 64)
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

// tile (c0, r0) of out[c][r] = in[r][c] for r < rows, zeros for r up to rows_pad
__device__ __forceinline__ void transpose_tile(bf16* t, const Source& in, int c0, int r0, bf16* out, int64_t ldo, int rows_pad) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 256 + threadIdx.x;
    const int c = (i & 7) * 8, r = i >> 3;
    to_lds(t, r, c, get8(in, r0 + r, c0 + c));
  }
  __syncthreads();
  put_transposed(t, out, ldo, r0, c0, in.cols, rows_pad);
}

// what gated_prepare_kernel makes, in tiles of 64 x 64: first the gradients of
// the projections, then the transposes
struct Prepare {
  Source dh, gate, up;  // [M][F]
  bf16* dgu;            // [M][2 Fp]
  bf16* dgut;           // [2 F][Mp]
  int Fp, Mp, tiles_g;
  Source in[3];         // X, and Wg, Wu or nothing
  bf16* out[3];
  int64_t ldo[3];
  int rows_pad[3], tiles[3];
};
template <int ACT>
__global__ void __launch_bounds__(256) gated_prepare_kernel(Prepare p) {
  __shared__ __attribute__((aligned(16))) bf16 tg[kTP * kTPitch], tu[kTP * kTPitch];
  int b = blockIdx.x;
  if (b >= p.tiles_g) {
    b -= p.tiles_g;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (b >= 0 && b < p.tiles[k]) {
        const int nc = cdiv(p.in[k].cols, kTP);
        transpose_tile(tg, p.in[k], b % nc * kTP, b / nc * kTP, p.out[k], p.ldo[k], p.rows_pad[k]);
      }
      b -= p.tiles[k];
    }
    return;
  }
  const int F = p.dh.cols, M = p.dh.rows, Fp = p.Fp, nf = cdiv(F, kTP);
  const int f0 = b % nf * kTP, m0 = b / nf * kTP;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 256 + threadIdx.x;
    const int c = (i & 7) * 8, r = i >> 3, m = m0 + r, f = f0 + c;
    bf16x8 vg = {}, vu = {};
    if (m < M && f < F) {
      const bf16x8 d8 = get8(p.dh, m, f), g8 = get8(p.gate, m, f), u8 = get8(p.up, m, f);
      float a[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float fv, dv;
        gate_slope<ACT>((float)g8[e], fv, dv);
        const float d = (float)d8[e];
        a[e] = f + e < F ? d * (float)u8[e] * dv : 0.f;
        u[e] = f + e < F ? d * fv : 0.f;
      }
      vg = cvt8(a);
      vu = cvt8(u);
    }
    if (m < M && f < Fp) {
      store8(p.dgu + (int64_t)m * 2 * Fp + f, vg);
      store8(p.dgu + (int64_t)m * 2 * Fp + Fp + f, vu);
    }
    to_lds(tg, r, c, vg);
    to_lds(tu, r, c, vu);
  }
  __syncthreads();
  put_transposed(tg, p.dgut, p.Mp, m0, f0, F, p.Mp);
  put_transposed(tu, p.dgut + (int64_t)F * p.Mp, p.Mp, m0, f0, F, p.Mp);
}

// dX of few rows, from the weights as they lie: part[s][m][d], the sum over
// K-blocks s, s + S, .. of 64 rows of Wg, then of Wu.
//
// A workgroup owns 128 columns d; a block of 64 f x 128 d goes to LDS as it is
// ([f][d], rows of 256 bytes) and is read across by ds_read_b64_tr_b16, which
// gives a lane four f of one d: MFMA fragments with K along f.  The
// rows of dG or dU beside it go to LDS once for the four waves.  Three images, one
// barrier a block: blocks b + 1 and b + 2 are on their way while b is multiplied.
// Slot s of LDS row r holds piece s ^ (2 (r & 3) + 8 (r >> 3 & 1)): the 8 rows that
// a read's 32 lanes touch fall on 8 different 32-byte ranges.
//
// Bound by the weights' bytes: 2 x 12288 x 4096 (201 MB) take 51 us with 1 row, 60
// with 128, 3.9 and 3.4 TB/s; a read of whole rows reaches 5.7.  Blocks of 256
// columns made it 49 and 62 (2 x 4096 x 1024: 14.4 us for 11.5), 2, 3 or 4 images
// and 1 to 4 workgroups a CU the same within 10 %.  With dG and dU from the caches
// into each wave's registers 128 rows took 135 us: 64 KB a block from the caches
// beside 16 KB of weights.
constexpr int kDxF = 64, kDxD = 128;
constexpr int kDxI = kDxD / 64;            // fragments of 16 columns a wave
constexpr int kDxRows = 2048 / kDxD;       // rows of weights that one load of the four waves covers
constexpr int kDxLoads = kDxF / kDxRows;
struct DxRows {
  const bf16* w[2];
  int64_t ldw;
  const bf16* dgu;
  int M, D, F, Fp;
  float* part;
};
// Two fragments of the weights, and the wait for them in the same block: before
// the builtin of such a read the compiler waits for the next block's loads too.
template <int OFF> __device__ __forceinline__ void weights(bf16x8 (&a)[2], const bf16* p0, const bf16* p1) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  s4 q[4];
  const uint32_t l0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) bf16*)p0;
  const uint32_t l1 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) bf16*)p1;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%6\n"
      "ds_read_b64_tr_b16 %1, %4 offset:%7\n"
      "ds_read_b64_tr_b16 %2, %5 offset:%6\n"
      "ds_read_b64_tr_b16 %3, %5 offset:%7\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3])
      : "v"(l0), "v"(l1), "n"(OFF), "n"(OFF + 2 * 4 * kDxD)
      : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i)
    a[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(q[2 * i], q[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7));
}
// 16 bytes a lane to LDS, from base (the wave's) + at (the lane's); a buffer load
// for the reason that Tile::run gives
__device__ __forceinline__ void to_image(const bf16* base, uint32_t at, bf16* lds) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(base), 0, -1, 0x27000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tile::lvoid*)lds, 16, at, 0, 0, 0);
}
template <int FB>
__global__ void __launch_bounds__(256) gated_dx_rows_kernel(DxRows p) {
  constexpr int kW = kDxF * kDxD, kX = 16 * FB * kDxF;  // elements of an image's two parts
  constexpr int kXLoads = FB / 2 + FB % 2;              // 32 rows a load of four waves
  constexpr int kAhead = 2;               // blocks on their way behind the one that is multiplied
  __shared__ __attribute__((aligned(128))) bf16 lds[(kAhead + 1) * (kW + kX)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int d0 = blockIdx.x * kDxD;
  const int nb = cdiv(p.F, kDxF);  // blocks a matrix
  const int S = gridDim.y, n = (2 * nb - (int)blockIdx.y + S - 1) / S;  // this split's blocks

  // load j of wave w: of the weights rows 16 j + 4 w + lane / 16, 16 pieces of 8
  // columns (past the end the last ones again); of dG | dU rows 32 j + 8 w + lane / 8
  auto swz = [](int r) { return 2 * (r & 3) + 8 * ((r >> 3) & 1); };
  uint32_t vw[kDxLoads], vx[kXLoads];
  const int lr = (wave * 64 + lane) / (kDxD / 8);
#pragma unroll
  for (int j = 0; j < kDxLoads; ++j)
    vw[j] = 2 * ((kDxRows * j + lr) * (uint32_t)p.ldw + min(8 * (lane % (kDxD / 8) ^ swz(kDxRows * j + lr)), p.D - 8 - d0));
#pragma unroll
  for (int j = 0; j < kXLoads; ++j) {
    const int m = 32 * j + 8 * wave + (lane >> 3);
    vx[j] = 2 * (min(m, p.M - 1) * 2 * (uint32_t)p.Fp + 8 * ((lane & 7) ^ (m & 7)));
  }
  auto load = [&](int b, bf16* img) {
    const int h = b >= nb, f0 = (b - h * nb) * kDxF;
    const bf16 *w = p.w[h] + (int64_t)f0 * p.ldw + d0, *x = p.dgu + h * p.Fp + f0;
#pragma unroll
    for (int j = 0; j < kDxLoads; ++j) {
      bf16* to = img + 2048 * j + 512 * wave;
      if (f0 + kDxF <= p.F || f0 + kDxRows * j + lr < p.F) to_image(w, vw[j], to);
      else to_image(reinterpret_cast<const bf16*>(tile::kZero16), 0, to);
    }
#pragma unroll
    for (int j = 0; j < kXLoads; ++j)
      if (FB > 1 || wave < 2) to_image(x, vx[j], img + kW + (32 * j + 8 * wave) * kDxF);
  };

  f32x4 acc[kDxI][FB];
#pragma unroll
  for (int i = 0; i < kDxI; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // a lane reads 4 columns of rows 8 g + r16 / 4 and 4 further
  int wat[kDxI];
#pragma unroll
  for (int i = 0; i < kDxI; ++i) {
    const int c = 16 * (kDxI * wave + i) + 4 * (r16 & 3), r = 8 * g + (r16 >> 2);
    wat[i] = r * kDxD + (((c >> 3) ^ swz(r)) << 3) + (c & 7);
  }
  for (int t = 0; t < min(n, kAhead); ++t) load(blockIdx.y + t * S, lds + t * (kW + kX));
  int at = 0;  // block b's image
  for (int t = 0; t < n; ++t) {
    const bf16* img = lds + at * (kW + kX);
    // block b is there, and every wave has read block b - 1 (a block whose rows end issues more
    // loads than these, in which case the wait is for more than block b)
    if (t + 1 < n) tile::vm_wait<kDxLoads + FB / 2>();
    else tile::vm_wait<0>();
    tile::barrier_raw();
    at = at == kAhead ? 0 : at + 1;
    if (t + kAhead < n) load(blockIdx.y + (t + kAhead) * S, lds + (at + kAhead - 1) % (kAhead + 1) * (kW + kX));
#pragma unroll
    for (int k = 0; k < kDxF / 32; ++k) {
      bf16x8 x[FB];
#pragma unroll
      for (int j = 0; j < FB; ++j) x[j] = load8(img + kW + (16 * j + r16) * kDxF + (((4 * k + g) ^ (r16 & 7)) << 3));
#pragma unroll
      for (int i = 0; i < kDxI; i += 2) {
        bf16x8 a[2];
        k == 0 ? weights<0>(a, img + wat[i], img + wat[i + 1]) : weights<2 * 32 * kDxD>(a, img + wat[i], img + wat[i + 1]);
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = mma(acc[i][j], a[0], x[j]);
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i + 1][j] = mma(acc[i + 1][j], a[1], x[j]);
      }
    }
  }
  // lane (r16, g): columns 4 g .. of fragment i, row r16 of group j
  float* out = p.part + (int64_t)blockIdx.y * p.M * p.D;
#pragma unroll
  for (int i = 0; i < kDxI; ++i) {
    const int d = d0 + 16 * (kDxI * wave + i) + 4 * g;
    if (d >= p.D) continue;  // (D is a multiple of 8)
#pragma unroll
    for (int j = 0; j < FB; ++j) {
      const int m = 16 * j + r16;
      if (m < p.M) *reinterpret_cast<f32x4*>(out + (int64_t)m * p.D + d) = acc[i][j];
    }
  }
}

// Products and sums that one launch does side by side: its workgroups are those
// of the first product, then of the second, then of the sums.
struct Product {
  Operands op;
  bf16* out;      // C[b][a], or
  float* part;    // S > 1: S partial sums of it over K
  int tiles, S, steps;  // K steps a split
};
// out = the sum of S partial arrays of n
struct Sum {
  const float* part;
  bf16* out;
  int64_t n;
  int S;
  __host__ __device__ int64_t blocks() const { return (n + 1023) / 1024; }
};
struct Work {
  Product p[2];
  Sum sum[2];
  __host__ __device__ int64_t products() const { return (int64_t)p[0].tiles * p[0].S + (int64_t)p[1].tiles * p[1].S; }
};

// values 1024 i .. of a sum, in order; eight partial arrays in flight (one after the
// other, 32 of 9 x 640 took 10 us)
__device__ __forceinline__ void sum_block(const Sum& q, int64_t block) {
  const int64_t n = q.n, i = (block * 256 + threadIdx.x) * 4;
  const float* part = q.part;
  if (i >= n) return;
  if (n % 4 == 0) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    for (; s + 8 <= q.S; s += 8) {
      f32x4 b[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) b[k] = *reinterpret_cast<const f32x4*>(part + (s + k) * n + i);
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += b[k][e];
    }
    for (; s < q.S; ++s) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(part + s * n + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += b[e];
    }
    *reinterpret_cast<bf16x4*>(q.out + i) = cvt4(a[0], a[1], a[2], a[3]);
  } else {
    for (int64_t e = i; e < std::min<int64_t>(i + 4, n); ++e) {
      float a = 0.f;
      for (int s = 0; s < q.S; ++s) a += part[s * n + e];
      q.out[e] = (bf16)a;
    }
  }
}
__device__ __forceinline__ void sums(const Work& w, int64_t block) {
  const int64_t n = w.sum[0].blocks();
  const int k = block >= n;
  sum_block(w.sum[k], block - k * n);
}
__global__ void __launch_bounds__(256) sums_kernel(Work w) { sums(w, blockIdx.x); }

template <int FA, int FB, class TO, class T>
__device__ __forceinline__ void put_tile(const T& t, char* lds, TO* out, int a0, int b0, const Operands& op) {
  const int wave = threadIdx.x >> 6, wa = wave >> 1, wb = wave & 1;
  const bool wide = op.arows % 8 == 0;
  typedef tile::RowStore<TO, FA, FA * FB >= 12 && sizeof(TO) == 2> Rows;  // (partial sums are read again at once)
  const Rows rows{lds + wave * Rows::kBytes};
  static_assert(4 * Rows::kBytes <= T::kLds, "row buffers fit the images");
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

// SUMS: products that are split into partial sums; of the largest tiles all or none
// are, both ways to store them would not fit the registers
enum Sums { kNone, kAll, kAny };
template <int FA, int FB, int KS, int NST, int WPE, Sums SUMS>
__global__ void __launch_bounds__(tile::kThreads, WPE) products_kernel(Work w) {
  typedef Tile<Bf16, FA, FB, KS, NST, false> T;
  __shared__ __attribute__((aligned(128))) char lds[T::kLds];
  int i = (int)blockIdx.x;
  const int n0 = w.p[0].tiles * w.p[0].S, n1 = w.p[1].tiles * w.p[1].S;
  if (i >= n0 + n1) {
    sums(w, i - n0 - n1);
    return;
  }
  const int second = i >= n0;
  const Product& p = w.p[second];
  i -= second * n0;
  const Operands op = p.op;
  const int split = i / p.tiles;
  int ta, tb;
  tile::tile_of(i - split * p.tiles, cdiv(op.arows, T::RA), cdiv(op.brows, T::RB), ta, tb);
  const int a0 = ta * T::RA, b0 = tb * T::RB;
  const int nk = (int)((op.kbytes + KS - 1) / KS);
  T t;
  t.run(op, lds, a0, b0, split * p.steps, min(nk, (split + 1) * p.steps));
  __syncthreads();  // every wave has read the last image
  if (SUMS == kAll || (SUMS == kAny && p.S > 1)) put_tile<FA, FB, float>(t, lds, p.part + (int64_t)split * op.arows * op.brows, a0, b0, op);
  else put_tile<FA, FB, bf16>(t, lds, p.out, a0, b0, op);
}

// outputs a workgroup, workgroups a CU, us a step (tile_gemm.h: Form).  640 x
// 16384 x 4096 150 / 126 / 103 / 101 / - / 92 us; 1024 x 8192 x 8192 216 / 176 / 133 /
// 113 / - / 157 us, the last in two sums over K 104; 4096 x 8192 x 64, all ends, 31 /
// 21 / 19 / 25 / - / 21; the fifth is for sizes that leave a last round of the others
// half empty: backward pass of 5578 x 1728 x 2880 270 us without it, 248 with
constexpr tile::Form kForms[] = {{64, 64, 2, 0.27f, 0.5f, 1.2f}, {128, 64, 2, 0.33f, 0.69f, 1.6f},
                                 {128, 128, 2, 0.55f, 1.15f, 2.9f}, {256, 128, 1, 0.86f, 0.86f, 4.8f},
                                 {256, 192, 1, 1.24f, 1.24f, 6.2f}, {256, 256, 1, 1.55f, 1.55f, 7.7f}};
constexpr int kNForms = 6;
// How the products are done: the form, and into how many sums over K each is split
// (where it has few tiles: 1024 x 777 outputs, K = 5472, 37.0 us in 56 tiles of 128
// x 128, 15.5 in 4 sums of them and 5 to add these up; 21.8 in 208 tiles of 64 x 64)
struct How {
  int form = 0, S[2] = {1, 1};
  float us = 1e30f;
};
struct Shape {
  int64_t arows, brows, kbytes;
  int64_t steps() const { return (kbytes + 127) / 128; }
};
// a launch of its own, and its tiles' start
constexpr float kLaunch = 4.f;
// adding sums up: 8 bytes a value of each
float join_us(const Shape& x, int S) { return S == 1 ? 0.f : (float)S * x.arows * x.brows * 8.f / 4e6f; }
// up to 16 sums of at least 4 steps
constexpr int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
bool splits(const Shape& x, int S) { return S == 1 || x.steps() / S >= 4; }

How how_alone(const Shape& x) {
  How best;
  for (int f = 0; f < kNForms; ++f) {
    const int64_t n = tile::workgroups(kForms[f], x.arows, x.brows);
    for (int S : kSplits) {
      if (!splits(x, S)) break;
      const float us = tile::form_us(kForms[f], n * S, (x.steps() + S - 1) / S) + join_us(x, S) + (S > 1 ? 7.f : 0.f);
      if (us < best.us) best = {f, {S, 1}, us};
    }
  }
  best.us += kLaunch;
  return best;
}
// Both products in one launch: none waits for the other's last tiles, and a launch
// and a join less.  Up to a round of the chip the longest workgroup counts, beyond it
// their sum and half a workgroup of the ones that end the launch.
How how_together(const Shape& x, const Shape& y) {
  How best;
  for (int f = 0; f < kNForms; ++f) {
    const tile::Form& t = kForms[f];
    const int64_t nx = tile::workgroups(t, x.arows, x.brows), ny = tile::workgroups(t, y.arows, y.brows);
    for (int S : kSplits) {
      if (!splits(x, S)) break;
      for (int R : kSplits) {
        if (!splits(y, R)) break;
        if (f == kNForms - 1 && (S == 1) != (R == 1)) continue;  // (products_kernel: SUMS)
        const float lx = (float)((x.steps() + S - 1) / S), ly = (float)((y.steps() + R - 1) / R);
        const float longest = std::max(lx, ly), shortest = std::min(lx, ly);
        const int64_t n = nx * S + ny * R, slots = (int64_t)tile::kCus * t.per_cu;
        float us = longest * (n <= tile::kCus ? t.one : t.full) + t.ends;
        if (n > slots)
          us = std::max(us, ((lx * t.full + t.ends) * (float)(nx * S) + (ly * t.full + t.ends) * (float)(ny * R)) / (float)slots +
                                0.5f * (shortest * t.full + t.ends));
        us += join_us(x, S) + join_us(y, R) + (S > 1 || R > 1 ? 7.f : 0.f);
        if (us < best.us) best = {f, {S, R}, us};
      }
    }
  }
  best.us += kLaunch;
  return best;
}

// dX from the weights as they are: for few rows, whole aligned pieces
bool dx_rows_fit(const GatedBwdParams& p) {
  const auto a = reinterpret_cast<uintptr_t>(p.wg) | reinterpret_cast<uintptr_t>(p.wu);
  return p.M <= 128 && p.D % 8 == 0 && p.ldw % 8 == 0 && p.ldw < (1 << 24) && a % 16 == 0;
}
// its K splits: about one workgroup a CU, at least two blocks each (71 rows,
// weights of 2 x 11520 x 3392: 46.8 us at one workgroup, 48.3 at two, 52.4 at four,
// and the partial sums' bytes grow with the splits)
int dx_rows_splits(int D, int F) {
  return std::max(1, std::min(cdiv(F, kDxF), tile::kCus / cdiv(D, kDxD)));
}

struct Plan {
  int M = 0, D = 0, F = 0;  // of this problem
  int Fp, Mp;
  Shape sx, sw;       // the products dX and dW
  How both, x, w;     // together (if that is faster: us), or one after the other
  int rows;           // K splits of dX by gated_dx_rows_kernel
  int64_t dgu, dgut, wt, xt, part[2], total;  // byte offsets
};
// (A training loop asks for the same plan again and again, twice a call: the last
// one is kept, 1.5 us a plan.)
const Plan& plan_of(int M, int D, int F) {
  static thread_local Plan q;
  if (q.M == M && q.D == D && q.F == F) return q;
  // rows of whole 128-byte lines: with rows of 7344 bytes every step's piece of a
  // row lies on two (640 x 17134 x 3672 140 us, of 8192 bytes in proportion 96)
  q.Fp = (int)round_up(F, 64);
  q.Mp = (int)round_up(M, 64);
  q.sx = {D, M, 4 * (int64_t)q.Fp};
  q.sw = {D, 2 * (int64_t)F, 2 * (int64_t)q.Mp};
  q.x = how_alone(q.sx);
  q.w = how_alone(q.sw);
  q.both = how_together(q.sx, q.sw);
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
  // dX of few rows from the weights as they are, or transposed beside dG and dU and
  // then in one launch with dW: one launch less, which short rows are worth (124 x 384 x
  // 704 17.8 -> 15.8 us)
  const float weights = 4.f * F * D;  // bytes
  const float as_they_are = kLaunch + std::max(2.5f, weights / 3.8e6f) + q.w.us, beside = q.both.us + 2.f * weights / 4e6f;
  q.rows = M <= 128 && as_they_are <= beside ? dx_rows_splits(D, F) : 0;
  const bool both = q.both.us < q.x.us + q.w.us;
  const int S = both ? q.both.S[0] : q.x.S[0], R = std::max(q.w.S[0], both ? q.both.S[1] : 1);
  q.part[0] = take(4 * (int64_t)std::max(S > 1 ? S : 0, q.rows) * M * D);
  q.part[1] = take(R > 1 ? 4 * R * 2 * (int64_t)F * D : 0);
  q.total = at;
  q.M = M;
  q.D = D;
  q.F = F;
  return q;
}

// out [brows][arows] = B A^T in the given form and splits
Product product(const char* a, const char* b, const Shape& x, bf16* out, float* part, int form, int S) {
  MCC_CHECK(x.kbytes <= (1 << 23), "gated_linear_bwd: row too long");
  Product p{};
  p.op.a[0] = p.op.a[1] = a;
  p.op.b = b;
  p.op.lda = p.op.ldb = x.kbytes;
  p.op.arows = (int)x.arows;
  p.op.brows = (int)x.brows;
  p.op.kbytes = x.kbytes;
  p.out = out;
  p.part = part;
  const int64_t n = tile::workgroups(kForms[form], x.arows, x.brows);
  MCC_CHECK(launchable(n * S, tile::kThreads), "gated_linear_bwd: too many rows");
  p.tiles = (int)n;
  p.steps = (int)((x.steps() + S - 1) / S);
  p.S = (int)((x.steps() + p.steps - 1) / p.steps);
  return p;
}

template <int FA, int FB, int NST, int WPE, Sums SUMS> void launch_tiles(const Work& w, hipStream_t s) {
  const int64_t n = w.products() + w.sum[0].blocks() + w.sum[1].blocks();
  MCC_CHECK(launchable(n, tile::kThreads), "gated_linear_bwd: too many rows");
  hipLaunchKernelGGL((products_kernel<FA, FB, 128, NST, WPE, SUMS>), dim3((unsigned)n), dim3(tile::kThreads), 0, s, w);
}
// the products and sums of w, then the sums of partial products
void run(const Work& w, int form, hipStream_t s) {
  if (form == 0) launch_tiles<1, 1, 4, 2, kAny>(w, s);
  else if (form == 1) launch_tiles<2, 1, 3, 2, kAny>(w, s);
  else if (form == 2) launch_tiles<2, 2, 2, 2, kAny>(w, s);
  else if (form == 3) launch_tiles<4, 2, 3, 1, kAny>(w, s);
  else if (form == 4) launch_tiles<4, 3, 2, 1, kAny>(w, s);
  else if (w.p[0].S == 1) launch_tiles<4, 4, 2, 1, kNone>(w, s);
  else launch_tiles<4, 4, 2, 1, kAll>(w, s);
  Work j{};
  for (int k = 0; k < 2; ++k)
    if (w.p[k].S > 1) j.sum[k] = {w.p[k].part, w.p[k].out, (int64_t)w.p[k].op.arows * w.p[k].op.brows, w.p[k].S};
  const int64_t n = j.sum[0].blocks() + j.sum[1].blocks();
  MCC_CHECK(launchable(n, 256), "gated_linear_bwd: too many rows");
  if (n > 0) hipLaunchKernelGGL(sums_kernel, dim3((unsigned)n), dim3(256), 0, s, j);
}

}  // namespace

namespace {
// sizes whose rows of the transposes a buffer load's offset reaches
void check_sizes(int M, int D, int F) {
  MCC_CHECK(M > 0 && D > 0 && F > 0, "gated_linear_bwd: empty problem");
  MCC_CHECK(M <= 4000000 && F <= (1 << 20), "gated_linear_bwd: too many rows");
}
}  // namespace

int64_t gated_backward_bytes(int M, int D, int F) {
  check_sizes(M, D, F);  // (before a workspace of that size is allocated)
  return plan_of(M, D, F).total;
}

void gated_backward(const GatedBwdParams& p, hipStream_t s) {
  check_sizes(p.M, p.D, p.F);
  MCC_CHECK(p.act >= GATE_NONE && p.act <= GATE_GELU, "gated_linear_bwd: unknown activation");
  MCC_CHECK(p.ldx >= p.D && p.ldw >= p.D, "gated_linear_bwd: row pitch");
  MCC_CHECK(reinterpret_cast<uintptr_t>(p.work) % 256 == 0, "gated_linear_bwd: workspace alignment");
  const Plan& q = plan_of(p.M, p.D, p.F);
  char* w = static_cast<char*>(p.work);
  bf16* dgu = reinterpret_cast<bf16*>(w + q.dgu);
  bf16* dgut = reinterpret_cast<bf16*>(w + q.dgut);
  bf16* wt = reinterpret_cast<bf16*>(w + q.wt);
  bf16* xt = reinterpret_cast<bf16*>(w + q.xt);
  float* part = reinterpret_cast<float*>(w + q.part[0]);
  float* partw = reinterpret_cast<float*>(w + q.part[1]);

  const bool rows = q.rows > 0 && dx_rows_fit(p);
  auto tiles = [](int r, int c) { return cdiv(r, kTP) * cdiv(c, kTP); };
  Prepare t;
  t.dh = source(p.dh, p.F, p.M, p.F);
  t.gate = source(p.gate, p.F, p.M, p.F);
  t.up = source(p.up, p.F, p.M, p.F);
  t.dgu = dgu; t.dgut = dgut;
  t.Fp = q.Fp; t.Mp = q.Mp;
  t.tiles_g = tiles(p.M, p.F);
  t.in[0] = source(p.x, p.ldx, p.M, p.D);
  t.in[1] = source(p.wg, p.ldw, p.F, p.D);
  t.in[2] = source(p.wu, p.ldw, p.F, p.D);
  t.out[0] = xt; t.ldo[0] = t.rows_pad[0] = q.Mp;
  t.out[1] = wt; t.out[2] = wt + q.Fp;
  t.ldo[1] = t.ldo[2] = 2 * q.Fp;
  t.rows_pad[1] = t.rows_pad[2] = q.Fp;
  t.tiles[0] = tiles(p.M, p.D);
  t.tiles[1] = t.tiles[2] = rows ? 0 : tiles(p.F, p.D);
  MCC_CHECK(launchable((int64_t)t.tiles_g + t.tiles[0] + t.tiles[1] + t.tiles[2], 256), "gated_linear_bwd: too many rows");
  const dim3 grid((unsigned)(t.tiles_g + t.tiles[0] + t.tiles[1] + t.tiles[2]));
  with_gate(p.act, [&](auto k) {
    hipLaunchKernelGGL((gated_prepare_kernel<decltype(k)::v>), grid, dim3(256), 0, s, t);
  });
  auto dx = [&](int form, int S) {
    return product(reinterpret_cast<const char*>(wt), reinterpret_cast<const char*>(dgu), q.sx, static_cast<bf16*>(p.dx), part,
                   form, S);
  };
  auto dw = [&](int form, int S) {
    return product(reinterpret_cast<const char*>(xt), reinterpret_cast<const char*>(dgut), q.sw, static_cast<bf16*>(p.dw), partw,
                   form, S);
  };
  if (rows) {
    const DxRows d{{static_cast<const bf16*>(p.wg), static_cast<const bf16*>(p.wu)}, p.ldw, dgu, p.M, p.D, p.F, q.Fp, part};
    const int S = q.rows;
    const dim3 g((unsigned)cdiv(p.D, kDxD), (unsigned)S);
    if (p.M <= 16) hipLaunchKernelGGL(gated_dx_rows_kernel<1>, g, dim3(256), 0, s, d);
    else if (p.M <= 32) hipLaunchKernelGGL(gated_dx_rows_kernel<2>, g, dim3(256), 0, s, d);
    else if (p.M <= 64) hipLaunchKernelGGL(gated_dx_rows_kernel<4>, g, dim3(256), 0, s, d);
    else hipLaunchKernelGGL(gated_dx_rows_kernel<8>, g, dim3(256), 0, s, d);
    Work k{};
    k.sum[0] = {part, static_cast<bf16*>(p.dx), (int64_t)p.M * p.D, S};
    k.p[0] = dw(q.w.form, q.w.S[0]);
    run(k, q.w.form, s);
  } else if (q.both.us < q.x.us + q.w.us) {
    // the longer workgroups first
    Work k{};
    k.p[0] = dx(q.both.form, q.both.S[0]);
    k.p[1] = dw(q.both.form, q.both.S[1]);
    if (k.p[0].steps < k.p[1].steps) std::swap(k.p[0], k.p[1]);
    run(k, q.both.form, s);
  } else {
    Work k{};
    k.p[0] = dx(q.x.form, q.x.S[0]);
    run(k, q.x.form, s);
    k.p[0] = dw(q.w.form, q.w.S[0]);
    run(k, q.w.form, s);
  }
  MCC_CHECK(hipGetLastError() == hipSuccess, "gated_linear_bwd: launch failed");
}

}  // namespace gpu
}  // namespace mcc

// Distillation loss and gradient from a teacher's top logits (feedforward.h:
// DistillParams).
//
// The gradient is a dense row p_j * scale T with at most K places where q is
// taken off.  A row is read once and written once: it stays in registers
// between (distill_row_kernel).  Sums and statistics are fp32; exponentials go
// to base 2 with log2(e) / T folded into one factor.  The K places are written
// a second time after the row's own stores have reached memory; of entries that
// name the same class the first writes, with the sum of them all in order, so
// the result does not depend on timing.
//
// Rows that do not fit the registers of a workgroup, and few long rows, which
// would leave most of the chip idle, are cut into chunks: one launch leaves
// every chunk's maximum and sum, a second joins them and writes the gradient,
// reading the logits again (distill_stat_kernel, distill_chunk_kernel).
#include "feedforward.h"
#include "mcc/common.h"
#include "mfma.h"

#include <algorithm>

namespace mcc {
namespace gpu {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// 8 logits as they came from memory.  (The compiler would keep bf16 logits
// widened, twice the registers; the empty asm in hide() makes it widen them
// again at each use.)
template <class T> struct Run;
template <> struct Run<bf16> {
  uint32_t w[4];
  __device__ __forceinline__ float operator[](int e) const { return ubits(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16); }
  __device__ __forceinline__ void hide() { asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3])); }
};
template <> struct Run<float> {
  float w[8];
  __device__ __forceinline__ float operator[](int e) const { return w[e]; }
  __device__ __forceinline__ void hide() {}
};

// elements j .. j+7 of a row of N, -inf where there is none; whole runs are
// 16-byte aligned (shift_of)
template <class T> __device__ __forceinline__ Run<T> get_run(const T* row, int j, int N) {
  Run<T> r;
  if (j >= 0 && j + 8 <= N) {
    r = __builtin_bit_cast(Run<T>, load8(row + j));
  } else {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = fbits(j + e >= 0 && j + e < N ? (float)row[j + e] : kNegInf);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[e] = b[2 * e] >> 16 | (b[2 * e + 1] & 0xffff0000u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.w[e] = ubits(b[e]);
    }
  }
  return r;
}
template <class T> __device__ __forceinline__ void put_run(T* row, int j, int N, bool aligned, const float (&v)[8]) {
  if (aligned && j >= 0 && j + 8 <= N) {
    if constexpr (sizeof(T) == 2) {
      const bf16x4 a = cvt4(v[0], v[1], v[2], v[3]), b = cvt4(v[4], v[5], v[6], v[7]);
      store8(row + j, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      store8(row + j, f32x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]});
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e >= 0 && j + e < N) row[j + e] = (T)v[e];
  }
}
// elements between the row's start and the 16-byte boundary before it: runs
// start at -shift, so that whole runs are aligned for any row length
template <class T> __device__ __forceinline__ int shift_of(const T* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}

// reductions over the RT threads of a row; `buf`: one value per wave of the
// block, free again after the next barrier of the caller
template <int RT, class F> __device__ __forceinline__ float row_reduce(float v, float* buf, F op) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = op(v, __shfl_xor(v, o));
  if constexpr (RT > 64) {
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = buf[0];
#pragma unroll
    for (int k = 1; k < RT / 64; ++k) v = op(v, buf[k]);
  }
  return v;
}
__device__ __forceinline__ float max_(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float add_(float a, float b) { return a + b; }

// A row's entries in LDS
struct Entries {
  int cls[kDistillMaxK];   // class, -1: not there
  float q[kDistillMaxK];   // q_k
  float lq[kDistillMaxK];  // log q_k
};

// Entry k of row m: its class (-1: not there) and logit
__device__ __forceinline__ int entry(const DistillParams& p, int64_t m, int k, float& t) {
  const int64_t at = m * p.K + k;
  const int64_t c = p.idx64 ? static_cast<const int64_t*>(p.idx)[at] : (int64_t) static_cast<const int32_t*>(p.idx)[at];
  t = p.t_f32 ? static_cast<const float*>(p.t)[at] : (float)static_cast<const bf16*>(p.t)[at];
  return c >= 0 && c < p.N && !(t == kNegInf) ? (int)c : -1;
}

// One wave: the teacher's distribution of row m into LDS.  Returns whether the
// row has entries.
__device__ __forceinline__ bool teacher(const DistillParams& p, int64_t m, Entries& s) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / p.temperature;
  float top = kNegInf;
  bool any = false;
  for (int k = lane; k < p.K; k += 64) {
    float t;
    const int cls = entry(p, m, k, t);
    s.cls[k] = cls;
    s.lq[k] = t;
    if (cls >= 0) {
      top = fmaxf(top, t);
      any = true;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (!__any(any)) return false;
  float sum = 0.f;
  for (int k = lane; k < p.K; k += 64) {
    const float e = s.cls[k] >= 0 ? exp2_((s.lq[k] - top) * c) : 0.f;
    s.q[k] = e;
    sum += e;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  const float ls = logf(sum);
  for (int k = lane; k < p.K; k += 64) {
    s.lq[k] = (s.lq[k] - top) / p.temperature - ls;
    s.q[k] /= sum;
  }
  return true;
}

// Of the row's entries k = t, t + nt, ..: the loss terms' sum, and the gradient
// at their classes within [lo, hi)
template <class TZ, class TG>
__device__ __forceinline__ float finish(const DistillParams& p, const Entries& s, const TZ* z, TG* dz, int t, int nt, int lo,
                                        int hi, float zmax, float zsum) {
  const float inv_t = 1.f / p.temperature, lz = logf(zsum), c = kLog2e / p.temperature;
  const float gs = p.scale * p.temperature / zsum, gq = p.scale * p.temperature;
  float loss = 0.f;
  for (int k = t; k < p.K; k += nt) {
    const int cls = s.cls[k];
    if (cls < 0) continue;
    const float zk = (float)z[cls];
    if (s.q[k] > 0.f || s.q[k] != s.q[k]) loss += s.q[k] * (s.lq[k] - ((zk - zmax) * inv_t - lz));
    if (!p.dz || cls < lo || cls >= hi) continue;
    float q = 0.f;
    bool first = true;
    for (int j = 0; j < p.K; ++j) {
      if (s.cls[j] == cls) {
        q += s.q[j];
        first = first && j >= k;
      }
    }
    if (first) dz[cls] = (TG)(exp2_((zk - zmax) * c) * gs - gq * q);
  }
  return loss;
}

// RT threads per row, NV runs of 8 logits per thread in registers
template <class TZ, class TG, int RT, int NV>
__global__ void __launch_bounds__(RT < 256 ? 256 : RT) distill_row_kernel(DistillParams p) {
  constexpr int kBlock = RT < 256 ? 256 : RT, kRows = kBlock / RT;
  __shared__ Entries ent[kRows];
  __shared__ float buf[3][kBlock / 64];
  __shared__ int some[kRows];
  const int t = threadIdx.x % RT, row = threadIdx.x / RT;
  const int64_t m = (int64_t)blockIdx.x * kRows + row;
  if (kRows > 1 && m >= p.M) return;  // (one wave per row: no barrier below is shared between rows)
  const int N = p.N;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  TG* dz = static_cast<TG*>(p.dz) + m * N;
  const int sh = shift_of(z);
  const bool aligned = reinterpret_cast<uintptr_t>(dz - sh) % 16 == 0;

  Run<TZ> zr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) zr[i] = get_run(z, 8 * (i * RT + t) - sh, N);
  Entries& en = ent[row];
  if (t < 64) {
    const bool h = teacher(p, m, en);
    if (t == 0) some[row] = h;
  }
  float zmax = kNegInf;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) zmax = fmaxf(zmax, zr[i][e]);
    zr[i].hide();
  }
  zmax = row_reduce<RT>(zmax, buf[0], max_);
  const float c = kLog2e / p.temperature;
  float zsum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) zsum += exp2_((zr[i][e] - zmax) * c);
    zr[i].hide();
  }
  zsum = row_reduce<RT>(zsum, buf[1], add_);
  const bool has = some[row];

  if (p.dz) {
    const float gs = has ? p.scale * p.temperature / zsum : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = has ? exp2_((zr[i][e] - zmax) * c) * gs : 0.f;
      put_run(dz, 8 * (i * RT + t) - sh, N, aligned, v);
    }
  }
  if (!has) {
    if (t == 0) p.loss[m] = 0.f;
    return;
  }
  // this wave's stores are in memory; behind the barrier, the whole row's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (RT > 64) __syncthreads();
  float loss = finish(p, en, z, dz, t, RT, 0, N, zmax, zsum);
  loss = row_reduce<RT>(loss, buf[2], add_);
  if (t == 0) p.loss[m] = loss * p.temperature * p.temperature;
}

constexpr int kChunk = 16384;  // logits per workgroup of the chunked form

// maximum and sum of exp2((z - maximum) log2(e) / T) of chunk blockIdx.y of row
// blockIdx.x
template <class TZ>
__global__ void __launch_bounds__(256) distill_stat_kernel(DistillParams p, float2* stat) {
  __shared__ float buf[2][4];
  const int64_t m = blockIdx.x;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  const int sh = shift_of(z), lo = (int)blockIdx.y * kChunk - sh;
  const float c = kLog2e / p.temperature;
  constexpr int NV = kChunk / (8 * 256);
  Run<TZ> zr[NV];
  float zmax = kNegInf, zsum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) zr[i] = get_run(z, lo + 8 * (i * 256 + (int)threadIdx.x), p.N);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) zmax = fmaxf(zmax, zr[i][e]);
    zr[i].hide();
  }
  zmax = row_reduce<256>(zmax, buf[0], max_);
  const float base = zmax == kNegInf ? 0.f : zmax;  // a chunk of -inf sums to 0
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) zsum += exp2_((zr[i][e] - base) * c);
  zsum = row_reduce<256>(zsum, buf[1], add_);
  if (threadIdx.x == 0) stat[m * gridDim.y + blockIdx.y] = make_float2(zmax, zsum);
}

// the gradient of chunk blockIdx.y of row blockIdx.x; chunk 0 leaves the loss
template <class TZ, class TG>
__global__ void __launch_bounds__(256) distill_chunk_kernel(DistillParams p, const float2* stat, int chunks) {
  __shared__ Entries en;
  __shared__ float buf[4];
  __shared__ int some;
  const int64_t m = blockIdx.x;
  const int N = p.N;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  TG* dz = static_cast<TG*>(p.dz) + m * N;
  const int sh = shift_of(z), lo = (int)blockIdx.y * kChunk - sh;
  const bool aligned = reinterpret_cast<uintptr_t>(dz - sh) % 16 == 0;
  const float c = kLog2e / p.temperature;
  if (threadIdx.x < 64) {
    const bool has = teacher(p, m, en);
    if (threadIdx.x == 0) some = has;
  }
  // the chunks' statistics in order
  float zmax = kNegInf, zsum = 0.f;
  for (int k = 0; k < chunks; ++k) zmax = fmaxf(zmax, stat[m * chunks + k].x);
  for (int k = 0; k < chunks; ++k) {
    const float2 s = stat[m * chunks + k];
    zsum += s.y * (s.x == kNegInf && zmax > kNegInf ? 0.f : exp2_((s.x - zmax) * c));
  }
  __syncthreads();
  const bool has = some;
  if (p.dz) {
    const float gs = has ? p.scale * p.temperature / zsum : 0.f;
    constexpr int NV = kChunk / (8 * 256);
#pragma unroll 4
    for (int i = 0; i < NV; ++i) {
      const int j = lo + 8 * (i * 256 + (int)threadIdx.x);
      const Run<TZ> r = get_run(z, j, N);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = has ? exp2_((r[e] - zmax) * c) * gs : 0.f;
      put_run(dz, j, N, aligned, v);
    }
  }
  if (!has) {
    if (blockIdx.y == 0 && threadIdx.x == 0) p.loss[m] = 0.f;
    return;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  float loss = finish(p, en, z, dz, (int)threadIdx.x, 256, std::max(lo, 0), std::min(lo + kChunk, N), zmax, zsum);
  if (blockIdx.y != 0) return;
  loss = row_reduce<256>(loss, buf, add_);
  if (threadIdx.x == 0) p.loss[m] = loss * p.temperature * p.temperature;
}

int chunks_of(int N) { return (int)ceil_div((int64_t)N + 7, kChunk); }  // (+ 7: the shift)

// the longest row (with its shift) that the registers of a workgroup hold
int row_limit(bool f32) { return f32 ? 1024 * 8 * 8 : 1024 * 8 * 16; }

// Few long rows: one workgroup per row would leave most CUs without one
bool chunked(int M, int N, bool f32) {
  return N + 7 > row_limit(f32) || (M < 128 && N > 2 * kChunk);
}

template <class TZ, class TG> void launch(const DistillParams& p, hipStream_t s) {
  constexpr bool f32 = sizeof(TZ) == 4;
  if (chunked(p.M, p.N, f32)) {
    const int n = chunks_of(p.N);
    float2* stat = static_cast<float2*>(p.work);
    const dim3 grid((unsigned)p.M, (unsigned)n);
    hipLaunchKernelGGL(distill_stat_kernel<TZ>, grid, dim3(256), 0, s, p, stat);
    hipLaunchKernelGGL((distill_chunk_kernel<TZ, TG>), p.dz ? grid : dim3((unsigned)p.M), dim3(256), 0, s, p, stat, n);
    return;
  }
  const int n = p.N + 7;
  auto rows = [&](int per) { return dim3((unsigned)ceil_div(p.M, per)); };
  if (n <= 64 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 64, 2>), rows(4), dim3(256), 0, s, p);
  else if (n <= 256 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 256, 2>), rows(1), dim3(256), 0, s, p);
  else if (n <= 256 * 8 * 4) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 256, 4>), rows(1), dim3(256), 0, s, p);
  else if (n <= 1024 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 2>), rows(1), dim3(1024), 0, s, p);
  else if (n <= 1024 * 8 * 4) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 4>), rows(1), dim3(1024), 0, s, p);
  else if (n <= 1024 * 8 * 8) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 8>), rows(1), dim3(1024), 0, s, p);
  else if constexpr (!f32) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 16>), rows(1), dim3(1024), 0, s, p);
}

}  // namespace

int64_t distill_bytes(int M, int N, bool z_f32) {
  return chunked(M, N, z_f32) ? (int64_t)sizeof(float2) * M * chunks_of(N) : 0;
}

void distill_kl(const DistillParams& p, hipStream_t s) {
  MCC_CHECK(p.M >= 0 && p.N > 0 && p.K >= 0, "distill_kl: empty rows");
  MCC_CHECK(p.N < (1 << 30), "distill_kl: too many classes");
  MCC_CHECK(p.K <= kDistillMaxK, "distill_kl: too many entries per row");
  MCC_CHECK(p.ldz >= p.N, "distill_kl: row pitch");
  MCC_CHECK(p.temperature > 0.f && p.temperature < __builtin_inff(), "distill_kl: temperature must be positive");
  MCC_CHECK(!p.z_f32 || p.dz_f32 || !p.dz, "distill_kl: a gradient of fp32 logits is fp32");
  MCC_CHECK(p.M == 0 || !chunked(p.M, p.N, p.z_f32) || p.work, "distill_kl: workspace missing");
  if (p.M == 0) return;
  if (p.z_f32) launch<float, float>(p, s);
  else if (p.dz_f32) launch<bf16, float>(p, s);
  else launch<bf16, bf16>(p, s);
  MCC_CHECK(hipGetLastError() == hipSuccess, "distill_kl: launch failed");
}

}  // namespace gpu
}  // namespace mcc

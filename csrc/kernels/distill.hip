// Distillation loss and gradient from a teacher's top logits (feedforward.h:
// DistillParams).
//
// The gradient is a dense row p_j * scale T with at most K places where q is
// taken off.  A row is read once and written once: it stays in registers
// between (distill_row_kernel).  Sums and statistics are fp32; exponentials go
// to base 2 with log2(e) / T folded into one factor.  Every thread keeps a
// running maximum and a sum relative to it, so the sum is formed while the
// logits still arrive and one exponential per logit is left for the gradient.
// The K places are written a second time by the wave that wrote their runs (a
// wave's stores are performed in order); of entries that name the same class
// the first writes, with the sum of them all in order, so the result does not
// depend on timing.
//
// Rows that do not fit the registers of a workgroup, and few long rows, which
// would leave most of the chip idle, are cut into chunks: one launch leaves
// every chunk's maximum and sum, a second joins them and writes the gradient,
// reading the logits again (distill_stat_kernel, distill_chunk_kernel).
//
// Bound by memory: 4096 x 120000 bf16 404 us, 1.97 GB at 4.9 TB/s (with stores past
// the caches 424); in chunks, where the logits come twice, 4096 x 151936 bf16 838
// (3.73 GB at 4.5), 2048 x 100000 fp32 539; 640 x 1000 fp32 6.4 us, a row's way in, two
// reductions and the way out.
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
  static __device__ __forceinline__ Run none() { return Run{{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}}; }
};
template <> struct Run<float> {
  float w[8];
  __device__ __forceinline__ float operator[](int e) const { return w[e]; }
  __device__ __forceinline__ void hide() {}
  static __device__ __forceinline__ Run none() {
    return Run{{kNegInf, kNegInf, kNegInf, kNegInf, kNegInf, kNegInf, kNegInf, kNegInf}};
  }
};

// Where the runs of a row of N lie: run v is elements 8 v - sh .., 16-byte
// aligned; first .. last are whole.  What is left, up to 7 elements at either
// end, goes to threads 0 .. 15 one by one (edge).
struct Grid {
  int sh, first, last;
  template <class T> __device__ __forceinline__ Grid(const T* row, int N) {
    sh = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    first = sh ? 1 : 0;
    last = max((N + sh) / 8 - 1, first - 1);
  }
  __device__ __forceinline__ bool whole(int v) const { return v >= first && v <= last; }
  // thread t's single element of a row of N, -1: none
  __device__ __forceinline__ int edge(int t, int N) const {
    const int e = t < 8 ? (sh && t < 8 - sh ? t : N) : t < 16 ? 8 * (last + 1) - sh + t - 8 : N;
    return e < N ? e : -1;
  }
};
// Runs v0 + i * step, i < NV, all in flight together; -inf for those that are
// not whole.  (The empty asm keeps the compiler from holding an address for
// each.)
template <class T, int NV>
__device__ __forceinline__ void get_runs(Run<T> (&r)[NV], const T* row, const Grid& g, int v0, int step) {
  if (g.last < g.first) {
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i] = Run<T>::none();
    return;
  }
  int v = v0;
#pragma unroll
  for (int i = 0; i < NV; ++i, v += step) {
    asm volatile("" : "+v"(v));
    const uint32_t at = (uint32_t)(8 * min(max(v, g.first), g.last) - g.sh) * (uint32_t)sizeof(T);
    r[i] = __builtin_bit_cast(Run<T>, load8(reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + at)));
  }
  v = v0;
#pragma unroll
  for (int i = 0; i < NV; ++i, v += step)
    if (!g.whole(v)) r[i] = Run<T>::none();
}

// Running maximum and sum of exp2((z - maximum) c).  The difference is taken
// before the factor: z c - maximum c in one fma would save an instruction and
// lose the difference's exactness (and its meaning, where the product
// overflows) for logits far from 0.
struct Soft {
  float top = kNegInf, sum = 0.f;
  template <class R> __device__ __forceinline__ void add(const R& r, float c) {
    float m = top;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, r[e]);
    const float base = m == kNegInf ? 0.f : m;  // (all -inf so far: every term is 0)
    float s = sum * exp2_((top - base) * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += exp2_((r[e] - base) * c);
    top = m;
    sum = s;
  }
  __device__ __forceinline__ void add_one(float z, float c) {
    if (z == kNegInf) return;
    const float m = fmaxf(top, z);
    sum = sum * exp2_((top - m) * c) + exp2_((z - m) * c);
    top = m;
  }
};

// The gradient without the entries' share, gs p, of the runs that get_runs took
// and of the single element: gs = 0: a row without entries
template <class TZ, class TG, int NV>
__device__ __forceinline__ void put_runs(Run<TZ> (&r)[NV], TG* dz, const Grid& g, int v0, int step, int edge, float ze, float c,
                                         float top, float gs) {
  const bool aligned = reinterpret_cast<uintptr_t>(dz - g.sh) % 16 == 0;
  int v = v0;
#pragma unroll
  for (int i = 0; i < NV; ++i, v += step) {
    asm volatile("" : "+v"(v));
    if (!g.whole(v)) continue;
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = gs == 0.f ? 0.f : exp2_((r[i][e] - top) * c) * gs;
    TG* q = reinterpret_cast<TG*>(reinterpret_cast<char*>(dz) + (int64_t)(8 * v - g.sh) * (int)sizeof(TG));
    if (aligned) {
      if constexpr (sizeof(TG) == 2) {
        const bf16x4 a = cvt4(d[0], d[1], d[2], d[3]), b = cvt4(d[4], d[5], d[6], d[7]);
        store8(q, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        store8(q, f32x8{d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7]});
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = (TG)d[e];
    }
  }
  if (edge >= 0) dz[edge] = (TG)(gs == 0.f ? 0.f : exp2_((ze - top) * c) * gs);
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

// A row's entries in LDS, K4 = K rounded up to 4 of each
struct Entries {
  int* cls;    // class, -1: not there
  float* q;    // q_k
  float* lq;   // log q_k
  float* zk;   // the student's logit
  float* sum;  // sum of q over the entries of this class; -1: not the first of them
  __device__ __forceinline__ Entries(char* lds, int row, int K4) {
    cls = reinterpret_cast<int*>(lds) + row * 5 * K4;
    q = reinterpret_cast<float*>(cls) + K4;
    lq = q + K4;
    zk = lq + K4;
    sum = zk + K4;
  }
};
__host__ __device__ __forceinline__ int entries_k4(int K) { return (K + 3) & ~3; }
__host__ __device__ __forceinline__ int entries_bytes(int K) { return 5 * 4 * entries_k4(K); }

// One wave: the teacher's distribution of row m (student's logits z) into LDS.
// Returns whether the row has entries.
template <class TZ> __device__ __forceinline__ bool teacher(const DistillParams& p, int64_t m, const TZ* z, const Entries& s) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / p.temperature;
  float top = kNegInf;
  bool any = false;
  for (int k = lane; k < entries_k4(p.K); k += 64) {
    int cls = -1;
    float t = 0.f;
    if (k < p.K) {
      const int64_t at = m * p.K + k;
      const int64_t i =
          p.idx64 ? static_cast<const int64_t*>(p.idx)[at] : (int64_t) static_cast<const int32_t*>(p.idx)[at];
      t = p.t_f32 ? static_cast<const float*>(p.t)[at] : (float)static_cast<const bf16*>(p.t)[at];
      if (i >= 0 && i < p.N && !(t == kNegInf)) cls = (int)i;
    }
    s.cls[k] = cls;
    s.lq[k] = t;
    s.zk[k] = cls >= 0 ? (float)z[cls] : 0.f;
    if (cls >= 0) {
      top = fmaxf(top, t);
      any = true;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  float sum = 0.f;
  for (int k = lane; k < entries_k4(p.K); k += 64) {
    const float e = s.cls[k] >= 0 ? exp2_((s.lq[k] - top) * c) : 0.f;
    s.q[k] = e;
    sum += e;
  }
  if (!__any(any)) return false;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  const float ls = logf(sum);
  for (int k = lane; k < p.K; k += 64) {
    s.lq[k] = (s.lq[k] - top) / p.temperature - ls;
    s.q[k] /= sum;
  }
  return true;
}

// Entries t, t + nt, ..: the sum of q over each one's class, by the first of them
__device__ __forceinline__ void join_classes(const Entries& s, int K, int t, int nt) {
  typedef int i4 __attribute__((ext_vector_type(4)));
  for (int k = t; k < K; k += nt) {
    const int cls = s.cls[k];
    float q = 0.f;
    bool first = cls >= 0;
    for (int j = 0; j < K; j += 4) {
      const i4 cj = *reinterpret_cast<const i4*>(s.cls + j);
      const f32x4 qj = *reinterpret_cast<const f32x4*>(s.q + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q += cj[e] == cls ? qj[e] : 0.f;
        first = first && !(cj[e] == cls && j + e < k);
      }
    }
    s.sum[k] = first ? q : -1.f;
  }
}

// One wave: the row's loss
__device__ __forceinline__ float row_loss(const DistillParams& p, const Entries& s, float ztop, float zsum) {
  const float inv_t = 1.f / p.temperature, lz = logf(zsum);
  float loss = 0.f;
  for (int k = threadIdx.x & 63; k < p.K; k += 64) {
    const float q = s.q[k];
    if (s.cls[k] >= 0 && !(q == 0.f)) loss += q * (s.lq[k] - ((s.zk[k] - ztop) * inv_t - lz));
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) loss += __shfl_xor(loss, o);
  return loss * p.temperature * p.temperature;
}

// One wave, after its runs of the gradient: the classes among them that have
// entries.  Of runs v0 .. v0 + runs - 1, v belongs to wave (v - v0) % RT / 64,
// single elements to wave 0.
template <int RT, class TG>
__device__ __forceinline__ void patch(const DistillParams& p, const Entries& s, TG* dz, const Grid& g, int v0, int runs, int wave,
                                      float ztop, float zsum) {
  const float c = kLog2e / p.temperature, gq = p.scale * p.temperature, gs = gq / zsum;
  // (the wave's stores above and below are performed in this order)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int k = threadIdx.x & 63; k < p.K; k += 64) {
    const int cls = s.cls[k];
    const float q = s.sum[k];
    const int v = (cls + g.sh) >> 3;
    if (cls >= 0 && !(q < 0.f) && v >= v0 && v < v0 + runs && (g.whole(v) ? (v - v0) % RT / 64 : 0) == wave)
      dz[cls] = (TG)(exp2_((s.zk[k] - ztop) * c) * gs - gq * q);
  }
}

// RT threads per row, NV runs of 8 logits per thread in registers
template <class TZ, class TG, int RT, int NV>
__global__ void __launch_bounds__(RT < 256 ? 256 : RT) distill_row_kernel(DistillParams p) {
  constexpr int kBlock = RT < 256 ? 256 : RT, kRows = kBlock / RT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float buf[2][kBlock / 64];
  __shared__ int some;
  const int t = threadIdx.x % RT, row = threadIdx.x / RT;
  const int64_t m = (int64_t)blockIdx.x * kRows + row;
  if (kRows > 1 && m >= p.M) return;  // (one wave per row: no barrier below is shared between rows)
  const int N = p.N;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  TG* dz = static_cast<TG*>(p.dz) + m * N;
  const Grid g(z, N);
  const float c = kLog2e / p.temperature;

  Run<TZ> zr[NV];
  get_runs(zr, z, g, t, RT);
  const int edge = g.edge(t, N);
  const float ze = edge >= 0 ? (float)z[edge] : kNegInf;
  const Entries en(lds, row, entries_k4(p.K));
  bool has = false;
  if (t < 64) {
    has = teacher(p, m, z, en);
    if (RT > 64 && t == 0) some = has;
  }
  Soft w;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    w.add(zr[i], c);
    zr[i].hide();
  }
  w.add_one(ze, c);
  const float top = row_reduce<RT>(w.top, buf[0], max_);
  w.sum *= w.top == kNegInf ? 0.f : exp2_((w.top - top) * c);
  join_classes(en, p.K, t, RT);
  const float sum = row_reduce<RT>(w.sum, buf[1], add_);
  if constexpr (RT > 64) has = some;

  if (t < 64) {
    const float loss = has ? row_loss(p, en, top, sum) : 0.f;
    if (t == 0) p.loss[m] = loss;
  }
  if (!p.dz) return;
  put_runs(zr, dz, g, t, RT, edge, ze, c, top, has ? p.scale * p.temperature / sum : 0.f);
  if (has) patch<RT>(p, en, dz, g, 0, NV * RT, t / 64, top, sum);
}

constexpr int kChunk = 16384;  // logits per workgroup of the chunked form

// thread t's single element where it lies in the chunk of the runs from v0 on
__device__ __forceinline__ int chunk_edge(const Grid& g, int v0, int t, int N) {
  const int e = g.edge(t, N), v = (e + g.sh) >> 3;
  return e >= 0 && v >= v0 && v < v0 + kChunk / 8 ? e : -1;
}

// maximum and sum of exp2((z - maximum) log2(e) / T) of chunk blockIdx.y of row
// blockIdx.x
template <class TZ>
__global__ void __launch_bounds__(256) distill_stat_kernel(DistillParams p, float2* stat) {
  __shared__ float buf[2][4];
  const int64_t m = blockIdx.x;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  const float c = kLog2e / p.temperature;
  constexpr int NV = kChunk / (8 * 256);
  Run<TZ> zr[NV];
  const Grid g(z, p.N);
  const int v0 = (int)blockIdx.y * (kChunk / 8);
  get_runs(zr, z, g, v0 + (int)threadIdx.x, 256);
  const int edge = chunk_edge(g, v0, (int)threadIdx.x, p.N);
  Soft w;
  w.add_one(edge >= 0 ? (float)z[edge] : kNegInf, c);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    w.add(zr[i], c);
    zr[i].hide();
  }
  const float top = row_reduce<256>(w.top, buf[0], max_);
  w.sum *= w.top == kNegInf ? 0.f : exp2_((w.top - top) * c);
  const float sum = row_reduce<256>(w.sum, buf[1], add_);
  if (threadIdx.x == 0) stat[m * gridDim.y + blockIdx.y] = make_float2(top, sum);
}

// the gradient of chunk blockIdx.y of row blockIdx.x; chunk 0 leaves the loss
template <class TZ, class TG>
__global__ void __launch_bounds__(256) distill_chunk_kernel(DistillParams p, const float2* stat, int chunks) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int some;
  const int64_t m = blockIdx.x;
  const int N = p.N, t = threadIdx.x;
  const TZ* z = static_cast<const TZ*>(p.z) + m * p.ldz;
  TG* dz = static_cast<TG*>(p.dz) + m * N;
  const Grid g(z, N);
  const int v0 = (int)blockIdx.y * (kChunk / 8);
  const float c = kLog2e / p.temperature;
  const Entries en(lds, 0, entries_k4(p.K));
  constexpr int NV = kChunk / (8 * 256);
  Run<TZ> zr[NV];
  if (p.dz) get_runs(zr, z, g, v0 + t, 256);
  const int edge = chunk_edge(g, v0, t, N);
  const float ze = edge >= 0 ? (float)z[edge] : kNegInf;
  if (t < 64) {
    const bool h = teacher(p, m, z, en);
    if (t == 0) some = h;
  }
  // the chunks' statistics in order
  float top = kNegInf, sum = 0.f;
  for (int k = 0; k < chunks; ++k) top = fmaxf(top, stat[m * chunks + k].x);
  for (int k = 0; k < chunks; ++k) {
    const float2 s = stat[m * chunks + k];
    sum += s.y * (s.x == kNegInf && top > kNegInf ? 0.f : exp2_((s.x - top) * c));
  }
  __syncthreads();
  const bool has = some;
  if (has) join_classes(en, p.K, t, 256);
  __syncthreads();
  if (blockIdx.y == 0 && t < 64) {
    const float loss = has ? row_loss(p, en, top, sum) : 0.f;
    if (t == 0) p.loss[m] = loss;
  }
  if (!p.dz) return;
  put_runs(zr, dz, g, v0 + t, 256, edge, ze, c, top, has ? p.scale * p.temperature / sum : 0.f);
  if (has) patch<256>(p, en, dz, g, v0, kChunk / 8, t / 64, top, sum);
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
    MCC_CHECK(launchable(p.M, 256, n), "distill_kl: too many rows");
    const dim3 grid((unsigned)p.M, (unsigned)n);
    hipLaunchKernelGGL(distill_stat_kernel<TZ>, grid, dim3(256), 0, s, p, stat);
    hipLaunchKernelGGL((distill_chunk_kernel<TZ, TG>), p.dz ? grid : dim3((unsigned)p.M), dim3(256),
                       entries_bytes(p.K), s, p, stat, n);
    return;
  }
  const int n = p.N + 7;
  MCC_CHECK(launchable(n <= 64 * 8 * 2 ? ceil_div(p.M, 4) : p.M, n <= 256 * 8 * 4 ? 256 : 1024), "distill_kl: too many rows");
  auto rows = [&](int per) { return dim3((unsigned)ceil_div(p.M, per)); };
  const int ent = entries_bytes(p.K);
  if (n <= 64 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 64, 2>), rows(4), dim3(256), 4 * ent, s, p);
  else if (n <= 256 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 256, 2>), rows(1), dim3(256), ent, s, p);
  else if (n <= 256 * 8 * 4) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 256, 4>), rows(1), dim3(256), ent, s, p);
  else if (n <= 1024 * 8 * 2) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 2>), rows(1), dim3(1024), ent, s, p);
  else if (n <= 1024 * 8 * 4) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 4>), rows(1), dim3(1024), ent, s, p);
  else if (n <= 1024 * 8 * 8) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 8>), rows(1), dim3(1024), ent, s, p);
  else if constexpr (!f32) hipLaunchKernelGGL((distill_row_kernel<TZ, TG, 1024, 16>), rows(1), dim3(1024), ent, s, p);
}

}  // namespace

int64_t distill_bytes(int M, int N, bool z_f32) {
  return chunked(M, N, z_f32) ? (int64_t)sizeof(float2) * M * chunks_of(N) : 0;
}

void distill_kl(const DistillParams& p, hipStream_t s) {
  MCC_CHECK(p.M >= 0 && p.N > 0 && p.K >= 0, "distill_kl: empty rows");
  MCC_CHECK(p.N <= (1 << 30) - (1 << 16), "distill_kl: too many classes");  // (65532 chunks)
  MCC_CHECK(p.K <= kDistillMaxK, "distill_kl: too many entries per row");
  MCC_CHECK(p.ldz >= p.N, "distill_kl: row pitch");
  MCC_CHECK(p.temperature >= 0.99e-6f && p.temperature <= 1.01e6f, "distill_kl: temperature out of range");
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

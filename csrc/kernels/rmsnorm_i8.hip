// RMS norm with the residual's addition and an 8-bit output with a scale per
// row (feedforward.h: RmsnormI8Params).
//
// One pass: a row's values stay in registers between its one read and its one
// write.  1 / rms is one positive factor of the whole row, so max |Y| is that
// factor times max |S W| and both reductions are of what is read, done in one
// round; Q = rint(S W * 127 / max |S W|) needs no 1 / rms at all.
// Statistics are fp32.  max is taken on the bits of |S W|, which order like the
// values with the infinities and NaN on top, so neither gets lost.
//
// Bound by memory: 16384 x 4096 with a residual, bf16 86-90 us, 470 MB at 5.2 to 5.5
// TB/s, fp32 155, 872 MB at 5.6; rows that are not whole 16-byte pieces by their single
// elements (16384 x 4095 bf16 189); one row of 4096 3.2 us, the row's way in, two
// barriers and the way out.
#include "feedforward.h"
#include "mcc/common.h"
#include "mfma.h"

namespace mcc {
namespace gpu {

namespace {

constexpr uint32_t kInfBits = 0x7f800000u;

template <class T> __device__ __forceinline__ void put_sum8(T* out, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const bf16x4 a = cvt4(v[0], v[1], v[2], v[3]), b = cvt4(v[4], v[5], v[6], v[7]);
    store8(out, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    store8(out, f32x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]});
  }
}

// RT threads per row, NV runs of 8 elements per thread; WIDE: rows, their
// pitches and D are whole 16-byte pieces, run i of thread t is elements
// 8 (i RT + t) ..; else single elements, (8 i + e) RT + t
template <class T, int RT, int NV, bool WIDE>
__global__ void __launch_bounds__(RT < 256 ? 256 : RT) rmsnorm_i8_kernel(RmsnormI8Params p) {
  constexpr int kBlock = RT < 256 ? 256 : RT;
  constexpr int kWaves = kBlock / 64;
  __shared__ float ss_part[kWaves];
  __shared__ uint32_t mx_part[kWaves];
  const int t = threadIdx.x % RT;
  const int64_t m = (int64_t)blockIdx.x * (kBlock / RT) + threadIdx.x / RT;
  const bool live = m < p.M;  // (RT < 256: the last block may hold rows that are not there)
  const T* x = static_cast<const T*>(p.x) + (live ? m : 0) * p.ldx;
  const T* r = p.r ? static_cast<const T*>(p.r) + (live ? m : 0) * p.ldr : nullptr;
  const T* w = static_cast<const T*>(p.w);
  T* sum = static_cast<T*>(p.sum) + m * p.D;
  const int D = p.D;

  float y[NV][8];
  float ss = 0.f;
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[8] = {}, g[8] = {};
    if constexpr (WIDE) {
      const int c = 8 * (i * RT + t);
      if (c < D) {
        const auto a = load8(x + c);
        const auto b = load8(w + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = (float)a[e];
          g[e] = (float)b[e];
        }
        if (r) {
          const auto d = load8(r + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += (float)d[e];
          if (live) put_sum8(sum + c, v);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = (8 * i + e) * RT + t;
        if (c < D) {
          v[e] = (float)x[c];
          g[e] = (float)w[c];
          if (r) {
            v[e] += (float)r[c];
            if (live) sum[c] = (T)v[e];
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss = fmaf(v[e], v[e], ss);
      y[i][e] = v[e] * g[e];
      mx = max(mx, fbits(y[i][e]) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    ss += __shfl_xor(ss, o);
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
  }
  if constexpr (RT > 64) {
    if ((threadIdx.x & 63) == 0) {
      ss_part[threadIdx.x >> 6] = ss;
      mx_part[threadIdx.x >> 6] = mx;
    }
    __syncthreads();
    ss = 0.f;
    mx = 0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      ss += ss_part[k];
      mx = max(mx, mx_part[k]);
    }
  }
  if (!live) return;
  // (with eps = 0 rstd is infinite for a row of zeros, or whose squares underflow)
  const float rstd = 1.f / sqrtf(ss / (float)D + p.eps);
  const bool good = ss < __builtin_inff() && mx < kInfBits && (mx == 0 || rstd < __builtin_inff());
  const float top = ubits(mx);
  // (127 / top overflows below 2^-121: such a row is scaled in two steps)
  const float up = top < 0x1p-100f ? 0x1p100f : 1.f;
  const float inv = good && mx ? 127.f / (top * up) : 0.f;
  if (t == 0) p.scale[m] = !good ? __builtin_nanf("") : mx ? top * rstd / 127.f : 0.f;
  int8_t* q = p.q + m * D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = good ? (uint32_t)(int)rintf(y[i][e] * up * inv) & 0xffu : 0u;
    if constexpr (WIDE) {
      const int c = 8 * (i * RT + t);
      if (c < D) {
        uint2 o;
        o.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        o.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
        *reinterpret_cast<uint2*>(q + c) = o;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = (8 * i + e) * RT + t;
        if (c < D) q[c] = (int8_t)b[e];
      }
    }
  }
}

template <class T, int RT, int NV> void launch(const RmsnormI8Params& p, bool wide, hipStream_t s) {
  constexpr int kBlock = RT < 256 ? 256 : RT;
  const int64_t n = ceil_div(p.M, kBlock / RT);
  MCC_CHECK(launchable(n, kBlock), "rmsnorm_i8: too many rows");
  const dim3 grid((unsigned)n);
  if (wide) hipLaunchKernelGGL((rmsnorm_i8_kernel<T, RT, NV, true>), grid, dim3(kBlock), 0, s, p);
  else hipLaunchKernelGGL((rmsnorm_i8_kernel<T, RT, NV, false>), grid, dim3(kBlock), 0, s, p);
}

template <class T> void pick(const RmsnormI8Params& p, hipStream_t s) {
  const int64_t v = 16 / (int64_t)sizeof(T);
  const auto a = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.r) | reinterpret_cast<uintptr_t>(p.w);
  const bool wide = p.D % 8 == 0 && a % 16 == 0 && p.ldx % v == 0 && (!p.r || p.ldr % v == 0);
  if (p.D <= 512) launch<T, 64, 1>(p, wide, s);
  else if (p.D <= 1024) launch<T, 64, 2>(p, wide, s);
  else if (p.D <= 2048) launch<T, 256, 1>(p, wide, s);
  else if (p.D <= 4096) launch<T, 256, 2>(p, wide, s);
  else if (p.D <= 8192) launch<T, 256, 4>(p, wide, s);
  else if (p.D <= 16384) launch<T, 1024, 2>(p, wide, s);
  else launch<T, 1024, 4>(p, wide, s);
}

}  // namespace

void rmsnorm_i8(const RmsnormI8Params& p, hipStream_t s) {
  MCC_CHECK(p.M >= 0 && p.D > 0, "rmsnorm_i8: empty rows");
  MCC_CHECK(p.D <= kRmsnormI8MaxD, "rmsnorm_i8: row too long");
  MCC_CHECK(p.ldx >= p.D && (!p.r || p.ldr >= p.D), "rmsnorm_i8: row pitch");
  MCC_CHECK((p.r == nullptr) == (p.sum == nullptr), "rmsnorm_i8: the sum goes with the residual");
  if (p.M == 0) return;
  if (p.f32) pick<float>(p, s);
  else pick<bf16>(p, s);
  MCC_CHECK(hipGetLastError() == hipSuccess, "rmsnorm_i8: launch failed");
}

}  // namespace gpu
}  // namespace mcc

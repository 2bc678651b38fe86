// One matrix-product tile loop for operands whose rows run along K, in units
// of bytes so that bf16 and 8-bit integers share it:
//
//   C[a][b] = sum_k A[a][k] B[b][k],   A [arows][K], B [brows][K]
//
// A is the side that runs along the output's contiguous axis: a lane ends with
// 16 consecutive A rows of one B row.
//
// The multiply is v_mfma_f32_32x32x16_bf16 or v_mfma_i32_32x32x32_i8: 32 cycles
// each on the same fragments, lane (r, g) = (lane & 31, lane >> 5) holding 16
// bytes of row r; a depth is 32 bytes of K, its lower half in g = 0.  A and B
// use the same map, so any order of K inside a depth cancels.  The 32 x 32 form
// reads half the operand registers per product of the 16 x 16 one, and its
// accumulators stay where they are (the compiler copied 180 of 256 registers a
// step around the 16 x 16 integer form).
//
// Workgroup: 4 waves in 2 x 2, wave tile (32 FA) x (32 FB), workgroup tile
// (64 FA) x (64 FB).  Operands go HBM -> LDS by buffer loads (16 bytes a
// lane) into NST images of KS bytes of K, image kt + NST into the place of image
// kt; how reads, loads and waits are dealt out among a step's MFMAs stands at
// `step` below.
//
// At 4 x 4 fragments a wave multiplies 2048 cycles per 128 bytes of K while the
// four waves read 128 KiB of LDS (1024 cycles at 128 B a cycle) and 64 KiB are
// written: the matrix unit is the longer side.  Eight waves of half the tile
// would read 192 KiB and be bound by LDS.
//
// Measured, 256 x 256 tiles over 8192 x 24576 x 4096 for half a second: bf16 1.50
// PFLOP/s, int8 2.78 Pop/s; a library's bf16 product of that size 1.59.  The clock gives
// way to power: with operands of zeros the same loop does 2.1 PFLOP/s and 4.0 Pop/s.  The
// matrix unit is busy 85 % of the cycles at 1.46 to 1.60 GHz in the product dX of
// gated_bwd.hip at 8192 x 4096 x 24576, whose stores are few.
//
// An LDS row of an image is KS bytes = KS/16 slots; slot s of row r holds the
// row's piece s ^ swz(r), applied on the source address of the load, so that
// the 16 rows that a read phase touches fall on 16 different 16-byte bank
// groups.  Row ρ of an A fragment is row 16 h + 4 q + e of the tile where
// ρ = 8 q + 4 h + e: the MFMA leaves rows 8 q + 4 h + e (q, e = 0..3) of its
// result in lane half h, which are then 16 consecutive rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mfma.h"

namespace mcc {
namespace gpu {
namespace tile {

typedef __attribute__((address_space(1))) void gvoid;
typedef __attribute__((address_space(3))) void lvoid;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;

// what a piece behind the end of K reads
__device__ __attribute__((aligned(64))) const uint32_t kZero16[16] = {0};

struct Bf16 {
  typedef bf16x8 frag;
  typedef f32x4 acc;  // 16 x 16 products (few_rows.h)
  typedef f32x16 acc32;
  static __device__ __forceinline__ acc mul(const frag& a, const frag& b, const acc& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ acc32 mul32(const frag& a, const frag& b, const acc32& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
struct I8 {
  typedef i32x4 frag;
  typedef i32x4 acc;
  typedef i32x16 acc32;
  static __device__ __forceinline__ acc mul(const frag& a, const frag& b, const acc& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ acc32 mul32(const frag& a, const frag& b, const acc32& c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};

// a[0] / a[1]: the sources of the tile's lower and upper A half (two matrices
// of the same shape and pitch) of a SPLIT tile, else a[0]
struct Operands {
  const char* a[2];
  const char* b;
  int64_t lda, ldb;  // row pitch in bytes (a multiple of 16, at most 2^23)
  int arows, brows;
  int64_t kbytes;    // bytes of K (a multiple of 16)
};

// Order of the tiles of a grid of na x nb: consecutive workgroups are dealt to
// the 8 XCDs in turn, so workgroup i works on position (i mod 8) * n/8 + i/8 of
// a walk over blocks of 8 B tiles: the 32 CUs of an XCD then hold about 8 x 4
// tiles and share those 12 operand tiles in their L2.
template <int G = 8>
__device__ __forceinline__ void tile_of(int i, int na, int nb, int& ta, int& tb) {
  const int n = na * nb;
  const int q = n >> 3, r = n & 7, x = i & 7;
  const int t = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (i >> 3);
  const int per = G * na;
  const int grp = t / per, in = t - grp * per;
  const int gb = min(G, nb - grp * G);
  ta = in / gb;
  tb = grp * G + (in - ta * gb);
}

// s_waitcnt with a count for one counter and the others left alone (vmcnt in
// bits 0-3 and 14-15, expcnt in 4-6, lgkmcnt in 8-11).  As a builtin, so that
// the compiler's own waits go on from it.
template <int N> __device__ __forceinline__ void vm_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0x0f70 | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void lds_read_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier_raw() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// SPLIT: the tile's A rows are two halves of 32 FA rows from a[0] and a[1] at
// the same place (a gate and its projection); every wave then owns FA/2
// fragments of each.  Otherwise wave row wa owns the 32 FA rows from 32 FA wa
// on.
template <class E, int FA, int FB, int KS, int NST, bool SPLIT>
struct Tile {
  static constexpr int RA = 64 * FA, RB = 64 * FB;
  static constexpr int kImage = (RA + RB) * KS;
  static constexpr int kLds = NST * kImage;
  static constexpr int kRowsPerLoad = 4096 / KS;  // rows that one load of the four waves covers
  static constexpr int JA = RA / kRowsPerLoad, JB = RB / kRowsPerLoad;
  static constexpr int kLoads = JA + JB;          // per thread and step
  static constexpr int kDepths = KS / 32;
  static constexpr int kReads = FA + FB;          // per depth
  static constexpr int kMuls = FA * FB;
  static_assert(KS == 128 || KS == 64, "image row");
  static_assert(!SPLIT || (FA % 2 == 0 && JA % 2 == 0), "both halves in whole fragments and loads");
  typedef typename E::frag frag;
  typedef typename E::acc32 acc_t;

  acc_t acc[FA][FB];

  // first A row (within the tile; within its half when SPLIT) of the 16 that
  // lane half h holds in fragment i
  static __device__ __forceinline__ int a_out(int wa, int i, int h) {
    return wa * (SPLIT ? RA / 4 : RA / 2) + 32 * (SPLIT ? i % (FA / 2) : i) + 16 * h;
  }
  static __device__ __forceinline__ int b_out(int wb, int j, int r) { return wb * (RB / 2) + 32 * j + r; }

  // K-steps [k0, k1) of the tile whose first rows are a0 (of each half's
  // source when SPLIT) and b0
  __device__ __forceinline__ void run(const Operands& p, char* lds, int a0, int b0, int k0, int k1) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, g = lane >> 5;
    const int wa = wave >> 1, wb = wave & 1;
    auto swz = [](int row) { return KS == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };

    // ---- image loads: load j of wave w covers rows from kRowsPerLoad j + (1024 / KS) w on ----
    constexpr int kSlots = KS / 16;
    const int lrow = wave * (1024 / KS) + lane / kSlots;
    const int piece = ((lane % kSlots) ^ swz(lrow)) * 16;  // the same for every j: kRowsPerLoad is a period of swz
    uint32_t va[JA], vb[JB];
#pragma unroll
    for (int j = 0; j < JA; ++j) {
      const int row = j * kRowsPerLoad + lrow - (SPLIT && j >= JA / 2 ? RA / 2 : 0);
      va[j] = (uint32_t)((int64_t)min(row, p.arows - 1 - a0) * p.lda) + piece;  // rows past the end: the last one again
    }
#pragma unroll
    for (int j = 0; j < JB; ++j)
      vb[j] = (uint32_t)((int64_t)min(j * kRowsPerLoad + lrow, p.brows - 1 - b0) * p.ldb) + piece;
    const char* pa0 = p.a[0] + (int64_t)a0 * p.lda;
    const char* pa1 = p.a[1] + (int64_t)a0 * p.lda;
    const char* pb = p.b + (int64_t)b0 * p.ldb;
    const int64_t kbytes = p.kbytes;
    // the operands' tiles as buffers: row offsets in a vector register, K in a scalar one
    const auto ra0 = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pa0), 0, -1, 0x27000);
    const auto ra1 = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pa1), 0, -1, 0x27000);
    const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pb), 0, -1, 0x27000);
    const auto rz = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(kZero16), 0, sizeof(kZero16), 0x27000);

    // load number j of step kt into the image at byte `at`; `tail`: the step may
    // run past the end of K, where both sides read zeros (one instruction more
    // in flight, so that a wait by count is only longer).  Buffer loads: for a
    // load through a global address the compiler, which cannot tell it from one
    // that may reach LDS, waits for ALL fragment reads wherever it has to wait
    // for one.
    auto load_one = [&](int kt, int at, int j, auto tail) {
      lvoid* img = (lvoid*)(lds + at + wave * 1024 + j * 4096);
      const bool is_a = j < JA, upper = SPLIT && j >= JA / 2;
      const auto r = is_a ? (upper ? ra1 : ra0) : rb;
      const uint32_t v = is_a ? va[is_a ? j : 0] : vb[is_a ? 0 : j - JA];
      if (!decltype(tail)::v || (int64_t)kt * KS + piece < kbytes)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, img, 16, v, kt * KS, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rz, img, 16, 0, 0, 0, 0);
    };
    auto load = [&](int kt, int at) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load_one(kt, at, j, ActK<1>{});
    };

    // ---- fragment reads: piece 2 d + g of depth d sits in slot (2 d + g) ^ swz(row) ----
    const int rho = 16 * ((r32 >> 2) & 1) + 4 * (r32 >> 3) + (r32 & 3);
    const int fa_at = (wa * (SPLIT ? RA / 4 : RA / 2) + rho) * KS + ((g ^ swz(rho)) << 4);
    const int fb_at = (RA + wb * (RB / 2) + r32) * KS + ((g ^ swz(r32)) << 4);
    frag fa[kDepths][FA], fb[kDepths][FB];
    // fragment t of the FB + FA of depth d
    auto read_one = [&](int at, int d, int t) {
      if (t < FB) {
        fb[d][t] = *reinterpret_cast<const frag*>(lds + at + (fb_at ^ (d << 5)) + t * 32 * KS);
      } else {
        const int i = t - FB;
        const int row = SPLIT ? (i >= FA / 2 ? RA / 2 : 0) + 32 * (i % (FA / 2)) : 32 * i;
        fa[d][i] = *reinterpret_cast<const frag*>(lds + at + (fa_at ^ (d << 5)) + row * KS);
      }
    };
    auto mul_one = [&](int d, int q) {
      acc[q / FB][q % FB] = E::mul32(fa[d][q / FB], fb[d][q % FB], acc[q / FB][q % FB]);
    };

#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

#pragma unroll
    for (int s = 0; s < NST; ++s)
      if (k0 + s < k1) load(k0 + s, s * kImage);
    if (k1 - k0 >= NST) vm_wait<(NST - 1) * kLoads>(); else vm_wait<0>();
    barrier_raw();
    int at = 0;  // image of step kt
#pragma unroll
    for (int t = 0; t < kReads; ++t) read_one(at, 0, t);

    // One step: kSlots MFMAs, with everything else dealt out among them by hand
    // (the source order, which the sched_barriers keep, is the schedule):
    //   first 3/8    reads of depths 1 ..
    //   half         barrier: every wave has read the image
    //   second half  loads of step kt + NST into its place
    //   7/8          wait for step kt + 1, barrier; then reads of its depth 0
    // Reads are bunched and loads spread because the two images must cover a
    // load's way to memory: an image is free for half a step more than if its
    // reads took the whole step, and a load every 64 cycles and wave is what the
    // address unit takes (16 cycles each): 16 in a quarter of the step stalled
    // the MFMAs behind them.
    constexpr int S = kDepths * kMuls, kB1 = S / 2, kB2 = S * 7 / 8, kR = (kDepths - 1) * kReads, kRS = (S * 3 + 7) / 8;
    constexpr int kBefore = (kB2 - kB1) * kLoads / (S - kB1);  // loads issued before the second wait
    auto mul_slot = [&](int s) {
      mul_one(s / kMuls, s % kMuls);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto read_slot = [&](int s) {
#pragma unroll
      for (int t = s * kR / kRS; t < (s + 1) * kR / kRS; ++t) read_one(at, 1 + t / kReads, t % kReads);
    };
    // mode 0: a load that lies wholly inside K; 1: one that may run past its
    // end; 2: no load
    auto step = [&](int kt, auto mode) {
      constexpr int kMode = decltype(mode)::v;
      const int next = at + kImage == kLds ? 0 : at + kImage;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s < kRS) read_slot(s);
        if (s == kB1) {
          lds_read_wait();
          barrier_raw();
        }
        if (s == kB2) {
          if (kMode < 2) vm_wait<(NST - 2) * kLoads + kBefore>(); else vm_wait<0>();
          barrier_raw();
        }
        if (kMode < 2 && s >= kB1) {
#pragma unroll
          for (int t = (s - kB1) * kLoads / (S - kB1); t < (s - kB1 + 1) * kLoads / (S - kB1); ++t)
            load_one(kt + NST, at, t, ActK<kMode>{});
        }
        if (s >= kB2) {
#pragma unroll
          for (int t = (s - kB2) * kReads / (S - kB2); t < (s - kB2 + 1) * kReads / (S - kB2); ++t) read_one(next, 0, t);
        }
        mul_slot(s);
      }
      at = next;
    };
    int kt = k0;
    const int kfull = min(k1, (int)(kbytes / KS)) - NST;  // steps whose load lies wholly inside K
    for (; kt < kfull; ++kt) step(kt, ActK<0>{});
    for (; kt + NST < k1; ++kt) step(kt, ActK<1>{});
    for (; kt + 1 < k1; ++kt) step(kt, ActK<2>{});
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < kRS) read_slot(s);
      mul_slot(s);
    }
  }
};

// 32 rows of an output (lane (r32, g) of a wave holds 16 consecutive columns of
// row r32 per fragment, NF fragments side by side) by way of LDS, so that a
// store instruction writes whole runs of a row: straight from the lanes it would
// write 32 rows in 16-byte pieces, and those quarter-line writes cost the int8
// product 20 % of its time at 8192 x 12288 x 4096.
//
// NT: stores that do not stay in the caches.  An output of a chip-filling
// product is larger than they are and would push out the operands that the
// other tiles still read: int8 8192 x 12288 x 4096 with inputs that change from
// call to call 349 -> 328 us (fp32 output 372 -> 348).
template <class TO, int NF, bool NT = false>
struct RowStore {
  static constexpr int kVec = 16 / (int)sizeof(TO);       // elements per 16-byte slot
  static constexpr int kSlots = 32 * NF / kVec;           // slots per row: 4, 8, 16 or 32
  static constexpr int kBytes = 32 * kSlots * 16;         // per wave
  char* lds;                                              // the wave's own kBytes

  static __device__ __forceinline__ int at(int row, int slot) { return (row * kSlots + (slot ^ (row & (kSlots - 1)))) * 16; }

  // fragment i's 16 columns of this lane
  __device__ __forceinline__ void put(int i, const float (&v)[16]) const {
    const int lane = threadIdx.x & 63, r32 = lane & 31, g = lane >> 5;
#pragma unroll
    for (int k = 0; k < 16 / kVec; ++k) {
      char* q = lds + at(r32, (32 * i + 16 * g) / kVec + k);
      if constexpr (sizeof(TO) == 2) {
        const bf16x4 a = cvt4(v[8 * k], v[8 * k + 1], v[8 * k + 2], v[8 * k + 3]);
        const bf16x4 b = cvt4(v[8 * k + 4], v[8 * k + 5], v[8 * k + 6], v[8 * k + 7]);
        *reinterpret_cast<bf16x8*>(q) = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        *reinterpret_cast<f32x4*>(q) = f32x4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
      }
    }
  }
  // the 32 rows to out[m0 ..][n0 ..] of an [M][N] matrix; wide: N is a
  // multiple of kVec (rows then start on 16 bytes and no slot straddles N)
  __device__ __forceinline__ void flush(TO* out, int m0, int n0, int M, int N, bool wide) const {
    const int lane = threadIdx.x & 63;
    if (wide) {
      constexpr int kRows = 64 / kSlots;  // rows per store (32 slots: two)
      const int slot = lane % kSlots, n = n0 + slot * kVec;
#pragma unroll
      for (int t = 0; t < 32 / kRows; ++t) {
        const int row = t * kRows + lane / kSlots, m = m0 + row;
        const f32x4 v = *reinterpret_cast<const f32x4*>(lds + at(row, slot));
        f32x4* q = reinterpret_cast<f32x4*>(out + (int64_t)m * N + n);
        if (m < M && n < N) {
          if constexpr (NT) __builtin_nontemporal_store(v, q);
          else *q = v;
        }
      }
    } else {
      // Rows that start anywhere: the 16-byte pieces of memory that lie wholly in
      // a row's run, each cut out of two slots, then the up to 15 bytes at either
      // end, an 8-, a 4- and a 2-byte store (with a store per value 777 x 1024 x
      // 2731 with three outputs took 24.0 us, so 22.3; rows of whole pieces 18.7).
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      typedef uint32_t u4 __attribute__((ext_vector_type(4)));
      typedef uint32_t u8 __attribute__((ext_vector_type(8)));
      constexpr int kRows = 64 / kSlots, kSize = (int)sizeof(TO);
      const int cols = min(32 * NF, N - n0);  // columns that exist
      if (cols <= 0) return;
      if (cols < kVec) {
        const int row = lane & 31;
        TO* q = out + (int64_t)(m0 + row) * N + n0;
        for (int c = lane >> 5; c < cols && m0 + row < M; c += 2)
          q[c] = *reinterpret_cast<const TO*>(lds + at(row, 0) + c * kSize);
        return;
      }
      auto skip = [&](int row) {  // columns before the first whole piece of a row
        const uintptr_t a = reinterpret_cast<uintptr_t>(out + (int64_t)(m0 + row) * N + n0);
        return (int)((16 - a % 16) % 16 / kSize);
      };
      // 16 bytes from byte `by` of lo on, into hi (whole vectors selected: an indexed array would be put into LDS)
      auto cut = [](const u4& lo, const u4& hi, int by) {
        u8 w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        w = by & 8 ? __builtin_shufflevector(w, w, 2, 3, 4, 5, 6, 7, 7, 7) : w;
        w = by & 4 ? __builtin_shufflevector(w, w, 1, 2, 3, 4, 5, 6, 7, 7) : w;
        u4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], by & 2);
        return v;
      };
      const int slot = lane % kSlots;
#pragma unroll 4
      for (int t = 0; t < 32 / kRows; ++t) {
        const int row = t * kRows + lane / kSlots, c0 = skip(row), c = c0 + slot * kVec;
        if (m0 + row >= M || c + kVec > cols) continue;
        const u4 lo = *reinterpret_cast<const u4*>(lds + at(row, slot));
        const u4 hi = *reinterpret_cast<const u4*>(lds + at(row, c0 ? slot + 1 : slot));
        *reinterpret_cast<u4*>(out + (int64_t)(m0 + row) * N + n0 + c) = cut(lo, hi, c0 * kSize);
      }
      // lane = (row, end): the piece that ends where the row's first whole one starts, or the one that
      // starts where the last ends, of which the run has the last or the first `len` values
      const int row = lane & 31, c0 = skip(row), n = (cols - c0) / kVec;
      const bool head = lane < 32;
      const int len = head ? c0 : cols - c0 - n * kVec;
      if (m0 + row >= M || len == 0) return;
      const int s = head ? 0 : n;  // (len > 0: a slot that exists)
      const u4 lo = *reinterpret_cast<const u4*>(lds + at(row, s));
      const u4 hi = *reinterpret_cast<const u4*>(lds + at(row, head ? 0 : min(s + 1, kSlots - 1)));
      const u4 v = cut(lo, hi, c0 * kSize);
      char* q = reinterpret_cast<char*>(out + (int64_t)(m0 + row) * N + n0 + c0 + (head ? -kVec : n * kVec));
      const int bytes = len * kSize;
      if (bytes & 8) *reinterpret_cast<u2*>(q + (head ? 8 : 0)) = head ? u2{v[2], v[3]} : u2{v[0], v[1]};
      if (bytes & 4) {
        const int d = head ? (bytes & 8 ? 1 : 3) : (bytes & 8 ? 2 : 0);
        *reinterpret_cast<uint32_t*>(q + 4 * d) = head ? (bytes & 8 ? v[1] : v[3]) : (bytes & 8 ? v[2] : v[0]);
      }
      if constexpr (kSize == 2) {
        if (len & 1) {  // value 8 - len (odd) or len - 1 (even)
          const int i = head ? 8 - len : len - 1;
          const uint32_t d = i & 4 ? (i & 2 ? v[3] : v[2]) : (i & 2 ? v[1] : v[0]);
          *reinterpret_cast<uint16_t*>(q + 2 * i) = (uint16_t)(head ? d >> 16 : d);
        }
      }
    }
  }
};

// ---- choice of a tile (host) ----
// A form of a product: workgroups of `rows_a` x `rows_b` outputs, `per_cu` of
// them to a CU, and, measured in us, what a step of 128 bytes of K takes, `one`
// while a CU holds one workgroup, `full` while it holds all `per_cu`, and what
// a workgroup's start and end take.
struct Form {
  int rows_a, rows_b, per_cu;
  float one, full, ends;
};
constexpr int kCus = 256;
inline int64_t workgroups(const Form& f, int64_t arows, int64_t brows) {
  return (arows + f.rows_a - 1) / f.rows_a * ((brows + f.rows_b - 1) / f.rows_b);
}
// n workgroups of `steps` steps: whole rounds of the chip, then what is left
inline float form_us(const Form& f, int64_t n, int64_t steps) {
  const int64_t slots = (int64_t)kCus * f.per_cu, rest = n % slots;
  const float us = n / slots * f.full + (rest == 0 ? 0.f : rest <= kCus ? f.one : f.full);
  return us * (float)steps + f.ends * (float)((n + slots - 1) / slots);
}
// the form that takes least
template <int N> inline int best_form(const Form (&f)[N], int64_t arows, int64_t brows, int64_t steps) {
  int best = 0;
  for (int i = 1; i < N; ++i)
    if (form_us(f[i], workgroups(f[i], arows, brows), steps) < form_us(f[best], workgroups(f[best], arows, brows), steps))
      best = i;
  return best;
}

}  // namespace tile
}  // namespace gpu
}  // namespace mcc

// Products of two bf16 matrices whose rows run along the summed axis:
// C[b][a] = sum_k A[a][k] B[b][k], float32 sums, a 256 x 256 tile of C a workgroup of
// eight wavefronts, 128 rows of A by 64 of B each: 32 results of 16 x 16 in 128
// registers, v_mfma_f32_16x16x32_bf16 (16 cycles).
//
// Steps of 64 values go to LDS without passing registers (16-byte direct loads, rows
// of 128 bytes an eight lanes), into a ring of five units of 32 KB, 64 values of 256
// rows of one operand each: the two in use, the other operand's next, and the two
// after. A wavefront reads half a step's fragments (12 ds_read_b128), then multiplies
// (32 MFMAs, 512 cycles), with a barrier after each; the wavefronts 4 to 7, one on
// each SIMD beside one of 0 to 3, run one barrier behind, so that a SIMD's matrix
// unit works for one of its two wavefronts while the other reads. A row's 16-byte
// chunk c lies at place c ^ (row mod 8): 16 lanes read from all banks (no conflicts
// counted). The loads for the steps to come are issued while reading and waited for
// with vmcnt(4), the youngest unit left in flight, two to three phases before use.
//
// Measured, 8192 x 32000 x 4096 with the loss's statistics behind it: 1.65 ms, 1,300
// TFLOP/s (the library's product of that shape with its bf16 result stored 1,360); a
// double buffer of both operands with one barrier a step 957; a ring of four stages of
// 32 values (rows of 64 bytes: twice the L2 requests) 1,260; four units released by
// halves of A's rows 1,286; the loads between the MFMAs 1,114, at their head 1,135.
// The clock falls to 1.65 GHz under this load; MFMAs are busy 64 to 70% of it.
//
// Small tiles, 128 x 128 by four wavefronts of 64 x 64 and two workgroups a CU, for
// products of few large ones: the same ring at half the size, one barrier a step; the
// other workgroup's wavefront fills a SIMD's pauses.
#pragma once

#include "common.h"

namespace cign {
namespace ntgemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;   // values of a row in LDS at a time; rows are a multiple of it
constexpr int kUnits = 5;   // LDS: a ring of kStep values of a tile's rows of A or of B

// A workgroup's tile of TA rows of A by TB of B, WA x WB wavefronts.
template <int TA_, int TB_, int WA_, int WB_>
struct Shape {
  static constexpr int TA = TA_, TB = TB_, WA = WA_, WB = WB_;
  static constexpr int kThreads = WA * WB * kWave;
  static constexpr int FA = TA / WA / 16, FB = TB / WB / 16;  // 16 x 16 results of a wavefront
  static constexpr bool kPaired = WA * WB == 8;               // two wavefronts a SIMD, in turn
  static constexpr int kUnitBytes = TA * kStep * 2;
  static constexpr int kLdsBytes = kUnits * kUnitBytes;
  static constexpr int kGroups = kPaired ? 1 : 2;             // workgroups a CU
  static_assert(TA == TB && TA == WA * WB * 32, "a wavefront brings 32 rows of each operand");
};
using Large = Shape<256, 256, 2, 4>;
using Small = Shape<128, 128, 2, 2>;

// Rows of bf16 values, ld values apart, 16-byte aligned, of a multiple of kStep
// values (zeros beyond their own); `part` values on lies the next part of values
// held in several (split float32).
struct Operand {
  const uint16_t* p;
  int64_t rows;
  int64_t ld;
  int64_t part;
};

// Place of a wavefront's results: four consecutive rows of A by one row of B a lane.
template <class S>
struct Place {
  int64_t a0, b0;
  __device__ Place(int ia, int ib) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
    a0 = static_cast<int64_t>(ia) * S::TA + (w % S::WA) * (S::TA / S::WA) + (l >> 4) * 4;
    b0 = static_cast<int64_t>(ib) * S::TB + (w / S::WA) * (S::TB / S::WB) + (l & 15);
  }
  __device__ __forceinline__ int64_t a(int fa) const { return a0 + fa * 16; }
  __device__ __forceinline__ int64_t b(int fb) const { return b0 + fb * 16; }
};

// Tile of workgroup id: workgroups go round the 8 XCDs, each of which takes a
// contiguous run of tiles, in bands of 8 tiles of B, tile of A by tile of A: the 32
// tiles at work on an XCD share 4 tiles of A and 8 of B in its L2.
__device__ __forceinline__ void tile_of(int id, int ta, int tb, int& ia, int& ib) {
  const int total = ta * tb, x = id & 7, k = id >> 3;
  const int each = total >> 3, more = total & 7;
  const int t = x * each + min(x, more) + k;
  const int band = t / (8 * ta), rest = t - band * 8 * ta;
  const int wide = min(8, tb - band * 8);
  ia = rest / wide;
  ib = band * 8 + rest % wide;
}

typedef __attribute__((address_space(1))) const void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// Which parts of A and B a segment multiplies, the smallest products first. A step's
// segments follow each other, since they share parts that the caches still hold (125
// rows against 126,733 classes of 1184 float32, gradients: 1.91 ms segment by segment,
// 1.71 so).
__device__ __forceinline__ int seg_a(int s) { return (0x001102 >> (4 * s)) & 0xF; }
__device__ __forceinline__ int seg_b(int s) { return (0x010120 >> (4 * s)) & 0xF; }

// The fragments of half a step from LDS, waited for in the same statement.
__device__ __forceinline__ void read_fragments(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[8], bf16x8 (&b)[4]) {
  asm volatile(
      "ds_read_b128 %0, %13\n"
      "ds_read_b128 %1, %13 offset:2048\n"
      "ds_read_b128 %2, %13 offset:4096\n"
      "ds_read_b128 %3, %13 offset:6144\n"
      "ds_read_b128 %4, %12\n"
      "ds_read_b128 %5, %12 offset:2048\n"
      "ds_read_b128 %6, %12 offset:4096\n"
      "ds_read_b128 %7, %12 offset:6144\n"
      "ds_read_b128 %8, %12 offset:8192\n"
      "ds_read_b128 %9, %12 offset:10240\n"
      "ds_read_b128 %10, %12 offset:12288\n"
      "ds_read_b128 %11, %12 offset:14336\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]),
        "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7])
      : "v"(at_a), "v"(at_b)
      : "memory");
}

__device__ __forceinline__ void read_fragments(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[4], bf16x8 (&b)[4]) {
  asm volatile(
      "ds_read_b128 %0, %9\n"
      "ds_read_b128 %1, %9 offset:2048\n"
      "ds_read_b128 %2, %9 offset:4096\n"
      "ds_read_b128 %3, %9 offset:6144\n"
      "ds_read_b128 %4, %8\n"
      "ds_read_b128 %5, %8 offset:2048\n"
      "ds_read_b128 %6, %8 offset:4096\n"
      "ds_read_b128 %7, %8 offset:6144\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3])
      : "v"(at_a), "v"(at_b)
      : "memory");
}

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The tile (ia, ib) of the product over ksteps steps, SEGS segments each; ends
// with a barrier behind the last use of lds. Rows past an operand's last repeat it:
// their results are not to be used.
template <class S, int SEGS>
__device__ __forceinline__ void product(const Operand& A, const Operand& B, int ia, int ib, int ksteps, char* lds,
                                        f32x4 (&acc)[S::FA][S::FB]) {
  constexpr int kUnitBytes = S::kUnitBytes;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
  const uint16_t* pa = A.p + static_cast<int64_t>(ia) * S::TA * A.ld;
  const uint16_t* pb = B.p + static_cast<int64_t>(ib) * S::TB * B.ld;
  const int ra = static_cast<int>(min(static_cast<int64_t>(S::TA), A.rows - static_cast<int64_t>(ia) * S::TA)) - 1;
  const int rb = static_cast<int>(min(static_cast<int64_t>(S::TB), B.rows - static_cast<int64_t>(ib) * S::TB)) - 1;
  uint32_t oa[4], ob[4];
  const int chunk = (l & 7) ^ (l >> 3);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = w * 32 + j * 8 + (l >> 3);
    oa[j] = static_cast<uint32_t>(min(r, ra)) * static_cast<uint32_t>(A.ld) + chunk * 8;
    ob[j] = static_cast<uint32_t>(min(r, rb)) * static_cast<uint32_t>(B.ld) + chunk * 8;
  }
  const int total = ksteps * SEGS;
  // the next unit of each operand: its step, the step in its segment, its segment
  int na = 0, ka = 0, ga = 0, nb = 0, kb = 0, gb = 0;
  int slot = 0;  // of the next unit
  const auto to_lds = [&](const uint16_t* src, const uint32_t (&o)[4]) {
    char* to = lds + slot * kUnitBytes + w * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_amdgcn_global_load_lds((GlobalPtr)(src + o[j]), (LdsPtr)(to + j * 1024), 16, 0, 0);
  };
  const auto next = [&](int& k, int& g) {
    if (++g == SEGS) {
      g = 0;
      ++k;
    }
    slot = slot == kUnits - 1 ? 0 : slot + 1;
  };
  const auto load_a = [&]() {
    if (na >= total) return;
    to_lds(pa + ka * kStep + (SEGS > 1 ? seg_a(ga) * A.part : 0), oa);
    next(ka, ga);
    ++na;
  };
  const auto load_b = [&]() {
    if (nb >= total) return;
    to_lds(pb + kb * kStep + (SEGS > 1 ? seg_b(gb) * B.part : 0), ob);
    next(kb, gb);
    ++nb;
  };
#pragma unroll
  for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
    for (int fb = 0; fb < S::FB; ++fb) acc[fa][fb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (total == 0) return;
  load_a();
  load_b();
  load_a();
  const int row = l & 15;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsPtr)lds)) + row * 128;
  const uint32_t at_a = base + (w % S::WA) * (S::TA / S::WA) * 128, at_b = base + (w / S::WA) * (S::TB / S::WB) * 128;
  const uint32_t half[2] = {static_cast<uint32_t>(((l >> 4) ^ (row & 7)) << 4),
                            static_cast<uint32_t>(((4 + (l >> 4)) ^ (row & 7)) << 4)};
  const bool second = S::kPaired && w >= 4;
  if (total > 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  barrier();
  if (second) barrier();
  uint32_t ua = 0, ub = kUnitBytes;  // units of this step
  for (int t = 0; t < total; ++t) {
    const bool more = t + 2 < total;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 a[S::FA], b[S::FB];
      if (h == 0) load_b();
      else load_a();
      read_fragments(at_a + ua + half[h], at_b + ub + half[h], a, b);
      if (h == 1 && second) {
        if (more) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      if (S::kPaired) {
        barrier();
        __builtin_amdgcn_s_setprio(1);
      }
#pragma unroll
      for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
        for (int fb = 0; fb < S::FB; ++fb)
          acc[fa][fb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[fa], b[fb], acc[fa][fb], 0, 0, 0);
      if (S::kPaired) __builtin_amdgcn_s_setprio(0);
      if (h == 1 && !second) {
        if (more) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      if (S::kPaired || h == 1) barrier();
    }
    ua = ua >= 3 * kUnitBytes ? ua - 3 * kUnitBytes : ua + 2 * kUnitBytes;
    ub = ub >= 3 * kUnitBytes ? ub - 3 * kUnitBytes : ub + 2 * kUnitBytes;
  }
  if (S::kPaired && !second) barrier();
  __syncthreads();
}

}  // namespace ntgemm
}  // namespace cign

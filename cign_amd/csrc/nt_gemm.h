// Products of two bf16 matrices whose rows run along the summed axis:
// C[b][a] = sum_k A[a][k] B[b][k], float32 sums, a 256 x 256 tile of C a workgroup.
#pragma once

#include "common.h"

namespace cign {
namespace ntgemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 256;                    // rows of A and of B of a workgroup's tile
constexpr int kStep = 64;                     // values of a row in LDS at a time
constexpr int kThreads = 512;
constexpr int kFragA = 8, kFragB = 4;         // 16 x 16 results of a wavefront: 128 rows of A, 64 of B
constexpr int kOperandBytes = kTile * kStep * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kLdsBytes = 2 * kStageBytes;

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
struct Place {
  int64_t a0, b0;
  __device__ Place(int ia, int ib) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
    a0 = static_cast<int64_t>(ia) * kTile + (w & 1) * 128 + (l >> 4) * 4;
    b0 = static_cast<int64_t>(ib) * kTile + (w >> 1) * 64 + (l & 15);
  }
  __device__ __forceinline__ int64_t a(int fa) const { return a0 + fa * 16; }
  __device__ __forceinline__ int64_t b(int fb) const { return b0 + fb * 16; }
};

// Tile of workgroup id: workgroups go round the 8 XCDs, each of which takes a
// contiguous run of tiles, in bands of 8 tiles of B, tile of A by tile of A.
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

// Which parts of A and B a segment multiplies, the smallest products first.
__device__ __forceinline__ int seg_a(int s) { return (0x001102 >> (4 * s)) & 0xF; }
__device__ __forceinline__ int seg_b(int s) { return (0x010120 >> (4 * s)) & 0xF; }

template <int SEGS>
__device__ __forceinline__ void product(const Operand& A, const Operand& B, int ia, int ib, int ksteps, char* lds,
                                        f32x4 (&acc)[kFragA][kFragB]) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
  const uint16_t* pa = A.p + static_cast<int64_t>(ia) * kTile * A.ld;
  const uint16_t* pb = B.p + static_cast<int64_t>(ib) * kTile * B.ld;
  const int ra = static_cast<int>(min(static_cast<int64_t>(kTile), A.rows - static_cast<int64_t>(ia) * kTile)) - 1;
  const int rb = static_cast<int>(min(static_cast<int64_t>(kTile), B.rows - static_cast<int64_t>(ib) * kTile)) - 1;
  uint32_t oa[4], ob[4];
  const int chunk = (l & 7) ^ (l >> 3);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = w * 32 + j * 8 + (l >> 3);
    oa[j] = static_cast<uint32_t>(min(r, ra)) * static_cast<uint32_t>(A.ld) + chunk * 8;
    ob[j] = static_cast<uint32_t>(min(r, rb)) * static_cast<uint32_t>(B.ld) + chunk * 8;
  }
  int seg = 0, k = 0;
  const auto load = [&](int stage) {
    const uint16_t* sa = pa + k * kStep;
    const uint16_t* sb = pb + k * kStep;
    if (SEGS > 1) {
      sa += seg_a(seg) * A.part;
      sb += seg_b(seg) * B.part;
    }
    char* to = lds + stage * kStageBytes + w * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __builtin_amdgcn_global_load_lds((GlobalPtr)(sa + oa[j]), (LdsPtr)(to + j * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((GlobalPtr)(sb + ob[j]), (LdsPtr)(to + kOperandBytes + j * 1024), 16, 0, 0);
    }
    if (++k == ksteps) {
      k = 0;
      ++seg;
    }
  };
#pragma unroll
  for (int fa = 0; fa < kFragA; ++fa)
#pragma unroll
    for (int fb = 0; fb < kFragB; ++fb) acc[fa][fb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int total = ksteps * SEGS;
  if (total > 0) load(0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int row = l & 15;
  const char* fa0 = lds + ((w & 1) * 128 + row) * 128;
  const char* fb0 = lds + kOperandBytes + ((w >> 1) * 64 + row) * 128;
  for (int t = 0; t < total; ++t) {
    const int off = (t & 1) * kStageBytes;
    bf16x8 a[2][kFragA], b[2][kFragB];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int slot = ((kk * 4 + (l >> 4)) ^ (row & 7)) * 16 + off;
#pragma unroll
      for (int f = 0; f < kFragB; ++f) b[kk][f] = *reinterpret_cast<const bf16x8*>(fb0 + f * 2048 + slot);
#pragma unroll
      for (int f = 0; f < kFragA; ++f) a[kk][f] = *reinterpret_cast<const bf16x8*>(fa0 + f * 2048 + slot);
    }
    if (t + 1 < total) load((t + 1) & 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int fa = 0; fa < kFragA; ++fa)
#pragma unroll
        for (int fb = 0; fb < kFragB; ++fb)
          acc[fa][fb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[kk][fa], b[kk][fb], acc[fa][fb], 0, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
}

}  // namespace ntgemm
}  // namespace cign

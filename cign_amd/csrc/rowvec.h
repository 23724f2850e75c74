// Rows of any width and alignment in 16-byte chunks: the accesses and the
// group reductions of the output operators (layernorm.hip, rowsoftmax.h).
//
// A row of n values is ceil(n / W) chunks of W values (W = 4 floats or 8
// bf16). Chunk c starts at value min(c * W, n - W): the last one of a ragged
// row overlaps the one before it, so every access is a whole chunk inside the
// row and only values at or past c * W belong to chunk c (`own`). Chunks past
// the last repeat it and own nothing, so loads need no branch. The vector
// types carry the alignment of one value: gfx950's 16-byte global accesses
// take any address, aligned ones at no cost, so odd widths and offset views
// need no kernel of their own. Rows of fewer than W values take W = 1.
#pragma once

#include "common.h"

namespace cign {
namespace rowvec {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Two floats rounded to bf16 (nearest even, NaN kept): v_cvt_pk_bf16_f32.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

template <typename T, int W>
struct RowChunk;

template <>
struct RowChunk<float, 4> {
  typedef float Raw __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ Raw load(const float* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ Raw load_past(const float* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p));
  }
  static __device__ __forceinline__ void unpack(const Raw& q, float (&v)[4]) {
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<Raw*>(p) = Raw{v[0], v[1], v[2], v[3]};
  }
  static __device__ __forceinline__ void store_past(float* p, const float (&v)[4]) {
    __builtin_nontemporal_store(Raw{v[0], v[1], v[2], v[3]}, reinterpret_cast<Raw*>(p));
  }
};

template <>
struct RowChunk<float, 8> {
  struct Raw {
    RowChunk<float, 4>::Raw a, b;
  };
  static __device__ __forceinline__ Raw load(const float* p) {
    return Raw{RowChunk<float, 4>::load(p), RowChunk<float, 4>::load(p + 4)};
  }
  static __device__ __forceinline__ void unpack(const Raw& q, float (&v)[8]) {
    v[0] = q.a.x; v[1] = q.a.y; v[2] = q.a.z; v[3] = q.a.w;
    v[4] = q.b.x; v[5] = q.b.y; v[6] = q.b.z; v[7] = q.b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    *reinterpret_cast<RowChunk<float, 4>::Raw*>(p) = RowChunk<float, 4>::Raw{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<RowChunk<float, 4>::Raw*>(p + 4) = RowChunk<float, 4>::Raw{v[4], v[5], v[6], v[7]};
  }
  static __device__ __forceinline__ void store_past(float* p, const float (&v)[8]) {
    __builtin_nontemporal_store(RowChunk<float, 4>::Raw{v[0], v[1], v[2], v[3]},
                                reinterpret_cast<RowChunk<float, 4>::Raw*>(p));
    __builtin_nontemporal_store(RowChunk<float, 4>::Raw{v[4], v[5], v[6], v[7]},
                                reinterpret_cast<RowChunk<float, 4>::Raw*>(p + 4));
  }
};

template <>
struct RowChunk<bf16, 8> {
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ Raw load(const bf16* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ Raw load_past(const bf16* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p));
  }
  static __device__ __forceinline__ void unpack(const Raw& q, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&v)[8]) {
    return Raw{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  }
  static __device__ __forceinline__ void store(bf16* p, const float (&v)[8]) { *reinterpret_cast<Raw*>(p) = pack(v); }
  static __device__ __forceinline__ void store_past(bf16* p, const float (&v)[8]) {
    __builtin_nontemporal_store(pack(v), reinterpret_cast<Raw*>(p));
  }
};

template <typename T>
struct RowChunk<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ Raw load_past(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const Raw& q, float (&v)[1]) { v[0] = to_f32(q); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) { *p = from_f32<T>(v[0]); }
  static __device__ __forceinline__ void store_past(T* p, const float (&v)[1]) { store(p, v); }
};

// Values per 16-byte chunk of T.
template <typename T>
constexpr int kChunk = 16 / sizeof(T);

// First value of chunk c of a row of n values (n >= W), and its first own
// value's place in the chunk (W or more: the chunk owns nothing).
template <int W>
__device__ __forceinline__ int chunk_start(int c, int n) {
  return min(c * W, n - W);
}

// ---------------------------------------------------------------------------
// Sums over the NT threads of a row: lanes of one wavefront (NT <= 64, a
// power of two, by butterflies) or the whole workgroup (NT = 256, 512, 1024:
// butterflies, then one LDS round). The LDS slots alternate between two sets,
// so one barrier a reduction is enough: a thread writes a set again only after
// the next reduction's barrier, which every reader of the former one passed.
// ---------------------------------------------------------------------------
template <int NT, int N>
struct GroupReduce {
  static constexpr int kWaves = NT / kWave;
  float (*slots)[N];  // [2][kWaves][N]
  int turn = 0;
  __device__ explicit GroupReduce(float (*s)[N]) : slots(s) {}

  __device__ __forceinline__ void sum(float (&v)[N]) {
    for_offsets<1, (NT < kWave ? NT : kWave)>([&](auto OC) {
      constexpr int o = decltype(OC)::value;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += xor_shfl<o>(v[i]);
    });
    if constexpr (NT > kWave) {
      float (*s)[N] = slots + turn * kWaves;
      if (lane_id() == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s[wave_id()][i] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = s[0][i];
#pragma unroll
      for (int k = 1; k < kWaves; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += s[k][i];
      turn ^= 1;
    }
  }
};

}  // namespace rowvec
}  // namespace cign

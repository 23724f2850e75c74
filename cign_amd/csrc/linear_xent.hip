// Cross entropy of a linear classifier over many classes, z = x W^T + b, by
// pieces of the classes, without keeping the logits:
//   lse = log sum_v e^(z_v), loss = lse - z_label,
//   dz_v = (g_loss + g_lse) e^(z_v - lse) - g_loss [v = label],
//   grad_x = dz W, grad_W = dz^T x, grad_b = sum over rows of dz.
//
// Forward: tiles of 256 rows by 256 classes (nt_gemm.h), or 128 by 128 where those
// leave CUs idle, whose largest logit and sum of exponentials a row leave the tile;
// join_kernel brings them together. Up to 64 rows, and more of float32 where that is
// faster, take no tiles: 64 classes a wavefront stream through LDS once for each 64 rows
// (stream_kernel, cut into runs of the summed axis where classes are few; few_kernel
// where rows do not start 16-byte aligned).
// Backward: the rows whose gradient is not zero are listed, a piece's logits are formed
// again, their gradient is stored in bf16 parts, and both products read it: the weight's
// with the rows as the summed axis, through LDS reads that turn 4 x 16 values.
//
// float32 operands are held as three bf16 parts of 8 bits each and multiplied in six
// products, the smallest first: the dropped ones lie below 2^-26 of a product, so the
// sums are float32's own. bfloat16 gradients of logits are rounded once, to bf16; the
// entry of a row's label, which holds most of its row's sum, has what that rounding
// dropped added back to the weight's gradient (Rests) and to the rows' (rows_out_kernel).
//
// What bounds it: the four products, 8 n V D operations, and beside them little. Forward
// and backward of 8192 rows, 32,000 classes, 4096 wide, a tenth of the rows without a
// label, 6.4 ms in bf16 (1,280 TFLOP/s over the four), of which 1.55 stats_kernel,
// 4 x 0.40 each of grad_kernel and the two out_kernels, 0.1 the rest; 4096 rows, 131,072
// classes, 2048 wide 7.2 ms. 24,492 rows, 2000 classes, 1280 wide, half of them without
// a label, float32: 1.7 ms (six products each: 1,300 TFLOP/s of bf16 inside the tiles).
// One row of 131,072 classes, 4096 wide, bf16: 185 us, 5.8 TB/s.
#include <algorithm>

#include "nt_gemm.h"
#include "rowvec.h"

namespace cign {
namespace xent {
using ntgemm::bf16x8;
using ntgemm::f32x4;
using ntgemm::kStep;
using ntgemm::Large;
using ntgemm::Operand;
using ntgemm::Place;
using ntgemm::Small;

constexpr int kMaxClasses = 1 << 20;
constexpr int kMaxWidth = 1 << 16;
constexpr int kMaxRows = 1 << 23;
constexpr int kFewRows = 64;
constexpr float kLog2e = 1.4426950408889634f;

template <int N>
using IC = std::integral_constant<int, N>;
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// e^d for d = z - m <= 0: relative error |d| 2^-24 and less.
__device__ __forceinline__ float exp_of(float d) { return exp2_of(d * kLog2e); }

// Two values as PARTS pairs of bf16 whose sums they are to 8 bits each. Parts below a
// value that is not finite are zero.
template <int PARTS>
__device__ __forceinline__ void split(float lo, float hi, uint32_t (&part)[PARTS]) {
  part[0] = rowvec::pack_bf16(lo, hi);
#pragma unroll
  for (int k = 1; k < PARTS; ++k) {
    lo -= __uint_as_float(part[k - 1] << 16);
    hi -= __uint_as_float(part[k - 1] & 0xffff0000u);
    part[k] = rowvec::pack_bf16(isfinite(lo) ? lo : 0.0f, isfinite(hi) ? hi : 0.0f);
  }
}

// A class's bias, of storage code `f32`.
__device__ __forceinline__ float bias_at(const void* bias, int f32, int64_t v) {
  return f32 ? static_cast<const float*>(bias)[v] : to_f32(static_cast<const bf16*>(bias)[v]);
}

// What the logits of a piece of classes are formed from.
struct Logits {
  Operand w, x;             // classes of the piece; rows
  int ksteps;
  const void* bias;         // of the whole vocabulary, or null
  int bias_f32;
  int64_t first;            // first class of the piece
  const int32_t* count;     // rows at work, on the device, or null for x.rows
  const int64_t* labels;
  __device__ __forceinline__ float bias_of(int64_t v) const {
    return bias ? bias_at(bias, bias_f32, first + v) : 0.0f;
  }
};

__device__ __forceinline__ int64_t thread_of() {
  return (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kBlock + threadIdx.x;
}

__device__ __forceinline__ int tiles(int64_t rows, int tile) { return static_cast<int>((rows + tile - 1) / tile); }

// (largest, sum of e^(value - largest)) of two sets
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float by = top == -INFINITY ? 0.0f : top;
  s = s * exp_of(m - by) + s2 * exp_of(m2 - by);
  m = top;
}

// Statistics of a tile: part[tile of classes][row], and the logit of each row's label.
template <class S, int SEGS>
__global__ __launch_bounds__(S::kThreads, S::kGroups) void stats_kernel(Logits f, int64_t n, float2* part, int first_tile,
                                                                    float* chosen) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  int ia, ib;
  ntgemm::tile_of(blockIdx.x, tiles(f.w.rows, S::TA), tiles(n, S::TB), ia, ib);
  f32x4 acc[S::FA][S::FB];
  ntgemm::product<S, SEGS>(f.w, f.x, ia, ib, f.ksteps, lds, acc);
  const Place<S> at(ia, ib);
  float2* red = reinterpret_cast<float2*>(lds);  // [WA][TB]
  const int wave = threadIdx.x / kWave, l = lane_id();
  const bool plain = !f.bias && (ia + 1) * S::TA <= f.w.rows;  // no class masked or behind the last
  float bias[S::FA][4];
  if (!plain)
#pragma unroll
    for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        bias[fa][r] = at.a(fa) + r < f.w.rows ? f.bias_of(at.a(fa) + r) : -INFINITY;
#pragma unroll
  for (int fb = 0; fb < S::FB; ++fb) {
    const int64_t row = at.b(fb);
    // the label's place behind the lane's first class
    const int64_t in = (f.labels && row < n ? f.labels[row] : -1) - f.first;
    const int want = in >= at.a0 && in < f.w.rows && in - at.a0 < S::TA / S::WA ? static_cast<int>(in - at.a0) : -1;
    float m = -INFINITY;
#pragma unroll
    for (int fa = 0; fa < S::FA; ++fa) {
      if (!plain)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[fa][fb][r] = bias[fa][r] == -INFINITY ? -INFINITY : acc[fa][fb][r] + bias[fa][r];
      const f32x4 z = acc[fa][fb];
      m = fmaxf(fmaxf(m, fmaxf(z[0], z[1])), fmaxf(z[2], z[3]));
      if ((want >> 4) == fa) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((want & 15) == r) chosen[row] = z[r];
      }
    }
    const float by = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
      for (int r = 0; r < 4; ++r) s += exp_of(acc[fa][fb][r] - by);
    join(m, s, xor_shfl<16>(m), xor_shfl<16>(s));
    join(m, s, xor_shfl<32>(m), xor_shfl<32>(s));
    if (l < 16) red[(wave % S::WA) * S::TB + (wave / S::WA) * (S::TB / S::WB) + fb * 16 + l] = make_float2(m, s);
  }
  __syncthreads();
  const int64_t row = static_cast<int64_t>(ib) * S::TB + threadIdx.x;
  if (threadIdx.x < S::TB && row < n) {
    float2 a = red[threadIdx.x];
    const float2 b = red[S::TB + threadIdx.x];
    join(a.x, a.y, b.x, b.y);
    part[static_cast<int64_t>(first_tile + ia) * n + row] = a;
  }
}

// Up to 64 rows: a wavefront takes 64 classes, four tiles of 16; values are fed to the
// matrix units in the order in which a lane's 16-byte chunks come, those of x alike.
// part[workgroup][row] as above.
template <typename T>
struct Few;
template <>
struct Few<bf16> {
  static constexpr int kLane = 8;  // values of a lane's chunk
  using Raw = bf16x8;
  static __device__ __forceinline__ f32x4 mul(const Raw& a, const Raw& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Few<float> {
  static constexpr int kLane = 4;
  using Raw = f32x4;
  static __device__ __forceinline__ f32x4 mul(const Raw& a, const Raw& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

template <typename T>
__device__ __forceinline__ typename Few<T>::Raw few_load(const T* p) {
  return __builtin_bit_cast(typename Few<T>::Raw, rowvec::RowChunk<T, Few<T>::kLane>::load(p));
}

// the values before `left` of a chunk, zeros behind
template <typename T>
__device__ __forceinline__ typename Few<T>::Raw few_tail(const T* p, int left) {
  T v[Few<T>::kLane];
#pragma unroll
  for (int i = 0; i < Few<T>::kLane; ++i) v[i] = i < left ? p[i] : from_f32<T>(0.0f);
  return __builtin_bit_cast(typename Few<T>::Raw, v);
}

constexpr int kFewClasses = 64;  // of a wavefront

// Statistics of a wavefront's classes from their products with n rows; part's sets of
// classes are `ldp` rows apart.
template <int TOKENS>
__device__ __forceinline__ void few_stats(f32x4 (&acc)[4][TOKENS / 16], int c0, int64_t n, int V, const void* bias,
                                          int bias_f32, const int64_t* labels, float2* part, int64_t ldp, float* chosen) {
  constexpr int TA = 4, TB = TOKENS / 16;
  const int l = lane_id();
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int64_t row = b * 16 + (l & 15);
    const int64_t want = labels && row < n ? labels[row] : -1;
    float m = -INFINITY;
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = c0 + a * 16 + (l >> 4) * 4 + r;
        float z = -INFINITY;
        if (v < V) {
          const float add = bias ? bias_at(bias, bias_f32, v) : 0.0f;
          if (add != -INFINITY) z = acc[a][b][r] + add;
          if (v == want) chosen[row] = z;
        }
        acc[a][b][r] = z;
        m = fmaxf(m, z);
      }
    const float by = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) s += exp_of(acc[a][b][r] - by);
    join(m, s, xor_shfl<16>(m), xor_shfl<16>(s));
    join(m, s, xor_shfl<32>(m), xor_shfl<32>(s));
    if (l < 16 && row < n) part[static_cast<int64_t>(c0 / kFewClasses) * ldp + row] = make_float2(m, s);
  }
}

// Rows of any alignment and width, read from where they lie into registers.
template <typename T, int TOKENS>
__global__ __launch_bounds__(kBlock) void few_kernel(int64_t n, int V, int D, const T* x, int64_t ldx, const T* w,
                                                     int64_t ldw, const void* bias, int bias_f32,
                                                     const int64_t* labels, float2* part, float* chosen) {
  using F = Few<T>;
  constexpr int L = F::kLane, TA = 4, TB = TOKENS / 16;
  const int l = lane_id();
  const int c0 = (blockIdx.x * kWavesPerBlock + wave_id()) * kFewClasses;
  if (c0 >= V) return;
  const int q = l >> 4;
  const T *wp[TA], *xp[TB];
#pragma unroll
  for (int i = 0; i < TA; ++i) wp[i] = w + static_cast<int64_t>(min(c0 + i * 16 + (l & 15), V - 1)) * ldw + q * L;
#pragma unroll
  for (int i = 0; i < TB; ++i) xp[i] = x + min(static_cast<int64_t>(i * 16 + (l & 15)), n - 1) * ldx + q * L;
  f32x4 acc[TA][TB];
#pragma unroll
  for (int a = 0; a < TA; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const auto steps = [&](auto UC, int k) {
    constexpr int U = decltype(UC)::value;
    typename F::Raw a[U][TA], b[U][TB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < TA; ++i) a[u][i] = few_load(wp[i] + k + u * 4 * L);
#pragma unroll
      for (int i = 0; i < TB; ++i) b[u][i] = few_load(xp[i] + k + u * 4 * L);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] = F::mul(a[u][i], b[u][j], acc[i][j]);
  };
  const int blocks = D / (16 * L), skew = blocks ? blockIdx.x * 13 % blocks : 0;
  for (int i = 0; i < blocks; ++i) steps(IC<4>(), (i + skew < blocks ? i + skew : i + skew - blocks) * 16 * L);
  int k = blocks * 16 * L;
  for (; k + 4 * L <= D; k += 4 * L) steps(IC<1>(), k);
  if (k < D) {
    typename F::Raw a[TA], b[TB];
    const int left = D - k - q * L;
#pragma unroll
    for (int i = 0; i < TA; ++i) a[i] = few_tail(wp[i] + k, left);
#pragma unroll
    for (int i = 0; i < TB; ++i) b[i] = few_tail(xp[i] + k, left);
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j) acc[i][j] = F::mul(a[i], b[j], acc[i][j]);
  }
  few_stats<TOKENS>(acc, c0, n, V, bias, bias_f32, labels, part, n, chosen);
}

// Four 16-byte reads of LDS, 2048 bytes apart, and one, waited for in the same statement.
__device__ __forceinline__ void read_four(uint32_t at, U32x4 (&v)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4\n"
      "ds_read_b128 %1, %4 offset:2048\n"
      "ds_read_b128 %2, %4 offset:4096\n"
      "ds_read_b128 %3, %4 offset:6144\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(at)
      : "memory");
}
__device__ __forceinline__ U32x4 read_one(uint32_t at) {
  U32x4 v;
  asm volatile("ds_read_b128 %0, %1\ns_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
  return v;
}

// A slot of the products of stream_kernel's workgroup x, run y of the steps.
template <int TOKENS>
__device__ __forceinline__ int64_t slot_of(int y, int x) {
  return (static_cast<int64_t>(y) * gridDim.x + x) * (4 * (TOKENS / 16) * kWave);
}

// Rows that start 16-byte aligned and are a multiple of 128 bytes wide: a workgroup is
// one wavefront; steps of 128 bytes of its 64 classes and of the rows of x go to LDS
// without passing registers, in a ring of steps. Nothing waits for another wavefront,
// and what finishes early makes room for the next. Each starts at another step, 13
// further on than the one before: rows of 8 KB read from their beginnings at the same
// time lie on few memory channels (one row against 131,072 x 4096 bf16: 186 us = 5.8
// TB/s, 218 from the beginning; float32 360 and 404). Two steps in the ring are
// enough for the memory (three 195 us, four 188). float32 rows beyond 16 are bounded
// by the matrix units, whose SIMDs have to have as many wavefronts each: rings, or
// room kept free, of 36 to 40 KB, four wavefronts a CU (40 rows: 640 us; five
// wavefronts a CU 1,010). More rows than TOKENS come in `groups`, workgroups `wide`
// apart (8: on one XCD) for the same classes. Few classes: the steps are cut into gridDim.y runs,
// whose products go to slots (slot_of), and few_join_kernel adds them up.
template <typename T, int TOKENS>
__global__ __launch_bounds__(kWave) void stream_kernel(int64_t n, int V, int D, const T* x, int64_t ldx, const T* w,
                                                       int64_t ldw, const void* bias, int bias_f32,
                                                       const int64_t* labels, float2* part, float* chosen, int groups, int wide,
                                                       f32x4* slots) {
  using F = Few<T>;
  constexpr int TB = TOKENS / 16;
  constexpr int kWide = 128 / sizeof(T);                    // values of a step
  constexpr int kStepBytes = (kFewClasses + TOKENS) * 128;
  constexpr int kLoads = 8 + 2 * TB;                        // of a step
  constexpr bool kBound = sizeof(T) == 4 && TOKENS > 16;    // by the matrix units
  constexpr int RING = kBound && TOKENS == 32 ? 3 : 2;
  constexpr int kRingBytes = RING * kStepBytes, kKept = kBound && kRingBytes < (33 << 10) ? 40 << 10 : kRingBytes;
  static_assert(kLoads * (RING - 1) < 63, "vmcnt");
  __shared__ __attribute__((aligned(1024))) char mine[kKept];
  const int l = lane_id();
  const int k = blockIdx.x / wide, set = k / groups * wide + blockIdx.x % wide, c0 = set * kFewClasses;
  if (c0 >= V) return;
  const int64_t first = static_cast<int64_t>(k % groups) * TOKENS, rows = min(static_cast<int64_t>(TOKENS), n - first);
  const int r8 = l >> 3, chunk = ((l & 7) ^ r8) * (16 / static_cast<int>(sizeof(T)));
  const T *wp[8], *xp[2 * TB];
#pragma unroll
  for (int j = 0; j < 8; ++j) wp[j] = w + static_cast<int64_t>(min(c0 + j * 8 + r8, V - 1)) * ldw + chunk;
#pragma unroll
  for (int j = 0; j < 2 * TB; ++j) xp[j] = x + (first + min(static_cast<int64_t>(j * 8 + r8), rows - 1)) * ldx + chunk;
  const int each = (D / kWide + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * each;
  const int total = min(each, D / kWide - begin);  // one at least
  const int skew = set * 13 % total;
  const auto load = [&](int step) {
    char* to = mine + (step % RING) * kStepBytes;
    const int t = begin + (step + skew < total ? step + skew : step + skew - total);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      __builtin_amdgcn_global_load_lds((ntgemm::GlobalPtr)(wp[j] + t * kWide), (ntgemm::LdsPtr)(to + j * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < 2 * TB; ++j)
      __builtin_amdgcn_global_load_lds((ntgemm::GlobalPtr)(xp[j] + t * kWide), (ntgemm::LdsPtr)(to + 8192 + j * 1024), 16,
                                       0, 0);
  };
  f32x4 acc[4][TB];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int t = 0; t < RING - 1 && t < total; ++t) load(t);
  const int row = l & 15;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((ntgemm::LdsPtr)mine)) + row * 128;
  for (int t = 0; t < total; ++t) {
    // what step t - 1 held was read and waited for
    if (t + RING - 1 < total) {
      load(t + RING - 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads * (RING - 1)) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const uint32_t from = base + (t % RING) * kStepBytes;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = from + (((4 * h + (l >> 4)) ^ (row & 7)) << 4);
      U32x4 a[4];
      read_four(at, a);
#pragma unroll
      for (int j = 0; j < TB; ++j) {
        const U32x4 b = read_one(at + 8192 + j * 2048);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[i][j] = F::mul(__builtin_bit_cast(typename F::Raw, a[i]), __builtin_bit_cast(typename F::Raw, b), acc[i][j]);
      }
    }
  }
  if (slots) {
    f32x4* to = slots + slot_of<TOKENS>(blockIdx.y, blockIdx.x) + l;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < TB; ++b) to[(a * TB + b) * kWave] = acc[a][b];
    return;
  }
  few_stats<TOKENS>(acc, c0, rows, V, bias, bias_f32, labels ? labels + first : nullptr, part + first, n, chosen + first);
}

// Statistics of stream_kernel's slots, summed in their order.
template <int TOKENS>
__global__ __launch_bounds__(kWave) void few_join_kernel(int64_t n, int V, const void* bias, int bias_f32,
                                                         const int64_t* labels, float2* part, float* chosen, int groups, int wide,
                                                         const f32x4* slots, int splits) {
  constexpr int TB = TOKENS / 16;
  const int k = blockIdx.x / wide, c0 = (k / groups * wide + blockIdx.x % wide) * kFewClasses;
  if (c0 >= V) return;
  const int64_t first = static_cast<int64_t>(k % groups) * TOKENS, rows = min(static_cast<int64_t>(TOKENS), n - first);
  f32x4 acc[4][TB];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (int y = 0; y < splits; ++y) {
    const f32x4* from = slots + slot_of<TOKENS>(y, blockIdx.x) + lane_id();
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < TB; ++b) acc[a][b] += from[(a * TB + b) * kWave];
  }
  few_stats<TOKENS>(acc, c0, rows, V, bias, bias_f32, labels ? labels + first : nullptr, part + first, n, chosen + first);
}

// loss and lse of ROWS rows a workgroup, 256 / ROWS threads a row over its nt tiles;
// the logarithm and the differences in float64, rounded once.
template <int ROWS>
__global__ __launch_bounds__(kBlock) void join_kernel(int64_t n, int V, int nt, const float2* part,
                                                      const int64_t* labels, int64_t ignore, const float* chosen,
                                                      float* loss, float* lse) {
  constexpr int kParts = kBlock / ROWS;
  __shared__ float2 red[kParts][ROWS];
  const int j = threadIdx.x % ROWS, k = threadIdx.x / ROWS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + j;
  float m = -INFINITY, s = 0.0f;
  if (row < n)
    for (int t = k; t < nt; t += kParts) {
      const float2 p = part[static_cast<int64_t>(t) * n + row];
      join(m, s, p.x, p.y);
    }
  red[k][j] = make_float2(m, s);
  __syncthreads();
  for (int h = kParts / 2; h > 0; h >>= 1) {
    if (k < h) {
      join(m, s, red[k + h][j].x, red[k + h][j].y);
      red[k][j] = make_float2(m, s);
    }
    __syncthreads();
  }
  if (k || row >= n) return;
  const double logs = log(static_cast<double>(s));
  lse[row] = static_cast<float>(static_cast<double>(m) + logs);
  if (!loss) return;
  const int64_t y = labels[row];
  float out = 0.0f;
  if (y != ignore) {
    if (y < 0 || y >= V)
      out = NAN;
    else if (s == 0.0f || chosen[row] == -INFINITY)
      out = isnan(s) ? NAN : INFINITY;
    else
      out = static_cast<float>(static_cast<double>(m) - static_cast<double>(chosen[row]) + logs);
  }
  loss[row] = out;
}

// Rows with a gradient, in order: list[0..count), and each row's place in it or -1;
// marks of the listed rows, their labels that are classes or -1, and rests of zero.
// One workgroup, 8192 rows at a time: a vote a wavefront for each 64 rows, the votes'
// counts added up in the rows' order.
__global__ __launch_bounds__(1024) void rows_kernel(int64_t n, const int64_t* labels, int64_t ignore,
                                                    const float* g_loss, const float* g_lse, int64_t V,
                                                    int32_t* list, int32_t* place, int32_t* count, int32_t* mark,
                                                    float* rest) {
  constexpr int kEach = 8, kWaves = 1024 / kWave;
  __shared__ int32_t sums[kEach * kWaves];
  int32_t base = 0;
  const uint64_t below = (1ull << lane_id()) - 1;
  for (int64_t b = 0; b < n; b += 1024 * kEach) {
    uint64_t votes[kEach];
    int64_t y[kEach];
    float g[kEach], h[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {  // every load before the first test
      const int64_t r = min(b + i * 1024 + threadIdx.x, n - 1);
      y[i] = g_loss ? labels[r] : 0;
      g[i] = g_loss ? g_loss[r] : 0.0f;
      h[i] = g_lse ? g_lse[r] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool on = b + i * 1024 + threadIdx.x < n && ((y[i] != ignore && g[i] != 0.0f) || h[i] != 0.0f);
      votes[i] = __ballot(on);
      if (lane_id() == 0) sums[i * kWaves + wave_id()] = __popcll(votes[i]);
    }
    __syncthreads();
    // sums[k]: rows before the 64 of vote k, in every wavefront's lanes two by two
    const int a = sums[2 * lane_id()], c = sums[2 * lane_id() + 1];
    int upto = a + c;
    for (int o = 1; o < kWave; o <<= 1) {
      const int t = __shfl_up(upto, o, kWave);
      if (lane_id() >= o) upto += t;
    }
    const int all = __shfl(upto, kWave - 1, kWave);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = i * kWaves + wave_id();
      const int before = __shfl(k & 1 ? upto - c : upto - a - c, k >> 1, kWave);
      const int64_t r = b + i * 1024 + threadIdx.x;
      const int at = base + before + __popcll(votes[i] & below);
      if (r < n) {
        const bool on = votes[i] >> lane_id() & 1;
        place[r] = on ? at : -1;
        if (on) {
          list[at] = static_cast<int32_t>(r);
          mark[at] = g_loss && y[i] != ignore && y[i] >= 0 && y[i] < V ? static_cast<int32_t>(y[i]) : -1;
          rest[at] = 0.0f;
        }
      }
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// Rows of D values of T as bf16 parts, Kp values apart with zeros behind the row's
// own, rows of a list where there is one; zeros for classes that a bias of -inf masks
// (their logits' gradients are zero, which a NaN would not stay).
template <typename T, int PARTS>
__global__ __launch_bounds__(kBlock) void pack_kernel(int64_t n, const int32_t* count, const int32_t* list, int D,
                                                      const T* src, int64_t ld, const void* bias, int bias_f32,
                                                      uint16_t* dst, int Kp, int64_t part) {
  const int64_t i = thread_of();
  const int per = Kp / 8;
  const int64_t r = i / per;
  const int c = static_cast<int>(i - r * per) * 8;
  if (r >= (count ? *count : n)) return;
  const T* row = src + (list ? list[r] : r) * ld;
  const bool on = !(bias && bias_at(bias, bias_f32, r) == -INFINITY);
  float v[8];
  if (on && c + 8 <= D) {
    rowvec::RowChunk<T, 8>::unpack(rowvec::RowChunk<T, 8>::load(row + c), v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = on && c + k < D ? to_f32(row[c + k]) : 0.0f;
  }
  U32x4 o[PARTS];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t p[PARTS];
    split<PARTS>(v[2 * k], v[2 * k + 1], p);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) o[q][k] = p[q];
  }
#pragma unroll
  for (int q = 0; q < PARTS; ++q) *reinterpret_cast<U32x4*>(dst + q * part + r * Kp + c) = o[q];
}

// Rows of D float32 values, `wide` apart with zeros behind their own.
__global__ __launch_bounds__(kBlock) void copy_kernel(int64_t n, int D, const float* src, int64_t ld, float* dst, int wide) {
  const int64_t i = thread_of();
  const int per = wide / 4;
  const int64_t r = i / per;
  const int c = static_cast<int>(i - r * per) * 4;
  if (r >= n) return;
  const float* row = src + r * ld;
  f32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = c + k < D ? row[c + k] : 0.0f;
  *reinterpret_cast<f32x4*>(dst + r * wide + c) = v;
}

// The gradient of a piece's logits, in bf16 parts: dz[row][class], zeros up to the next
// multiple of kStep of each axis; and the tile's sums over its rows, for the bias.
struct Grads {
  const int32_t* list;
  const float* lse;
  const float* g_loss;     // null: none
  const float* g_lse;      // null: none
  int64_t ignore;
  int64_t V;
  uint16_t* dz;
  int64_t ld, part;
  float* bias_part;        // [tile of rows][class of the piece] or null
  float* rest;             // what rounding to bf16 leaves of the label's entry, by row
};

// A tile of 16-bit values in LDS, rows of 512 (256) bytes and 16 more, so that
// neither a column's nor a row's accesses meet on few banks.
template <class S>
constexpr int kStageRow = S::TA * 2 + 16;
static_assert(Large::TB * kStageRow<Large> <= Large::kLdsBytes && Small::TB * kStageRow<Small> <= Small::kLdsBytes,
              "a tile of results fits the operands' LDS");

// Writes the staged tile to global rows `ld` values apart, 16 bytes a lane: rows below `rows`, values below `cols` (of the tile), chunks whole where cols
// is a multiple of 8, value by value at a ragged end.
template <class S, bool RAGGED>
__device__ __forceinline__ void store_tile(const char* lds, uint16_t* out, int64_t ld, int rows, int cols) {
  typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
  constexpr int kLanes = S::TA / 8;
  const int c = (threadIdx.x % kLanes) * 8;
#pragma unroll 4
  for (int r = threadIdx.x / kLanes; r < S::TB; r += S::kThreads / kLanes) {
    if (r >= rows || c >= cols) continue;
    const U32x4 v = *reinterpret_cast<const U32x4*>(lds + r * kStageRow<S> + c * 2);
    uint16_t* to = out + r * ld + c;
    if (!RAGGED) {
      *reinterpret_cast<U32x4*>(to) = v;
    } else if (c + 8 <= cols) {
      *reinterpret_cast<Any*>(to) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < cols) to[i] = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Stages four consecutive rows of A by one of B a lane: [row of B][row of A].
template <class S>
__device__ __forceinline__ void stage(char* lds, int fa, int fb, uint32_t first, uint32_t second) {
  const int w = threadIdx.x / kWave, l = lane_id();
  *reinterpret_cast<uint2*>(lds + ((w / S::WA) * (S::TB / S::WB) + fb * 16 + (l & 15)) * kStageRow<S> +
                            ((w % S::WA) * (S::TA / S::WA) + fa * 16 + (l >> 4) * 4) * 2) = make_uint2(first, second);
}

template <class S, int SEGS>
__global__ __launch_bounds__(S::kThreads, S::kGroups) void grad_kernel(Logits f, Grads g) {
  constexpr int PARTS = SEGS > 1 ? 3 : 1;
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  const int64_t n = *f.count;
  const int ta = tiles(f.w.rows, S::TA), tb = tiles(n, S::TB);
  if (static_cast<int64_t>(blockIdx.x) >= static_cast<int64_t>(ta) * tb) return;
  int ia, ib;
  ntgemm::tile_of(blockIdx.x, ta, tb, ia, ib);
  f32x4 acc[S::FA][S::FB];
  Operand x = f.x;
  x.rows = n;
  ntgemm::product<S, SEGS>(f.w, x, ia, ib, f.ksteps, lds, acc);
  const Place<S> at(ia, ib);
  const int wave = threadIdx.x / kWave, l = lane_id();
  const int rows = static_cast<int>(min(static_cast<int64_t>(S::TB), n - static_cast<int64_t>(ib) * S::TB));
  const int classes = static_cast<int>(min(static_cast<int64_t>(S::TA), f.w.rows - static_cast<int64_t>(ia) * S::TA));
  const int a0 = (wave % S::WA) * (S::TA / S::WA) + (l >> 4) * 4;  // the lane's first class in the tile
  float own[S::FB], all[S::FB], shift[S::FB];
  int want[S::FB];  // the label's place behind the lane's first class
#pragma unroll
  for (int fb = 0; fb < S::FB; ++fb) {
    const int64_t row = at.b(fb);
    own[fb] = all[fb] = 0.0f;
    shift[fb] = INFINITY;  // e^(z - inf) = 0
    want[fb] = -1;
    if (row < n) {
      const int64_t src = g.list[row];
      const int64_t y = f.labels ? f.labels[src] : g.ignore;
      if (y != g.ignore && g.g_loss) {
        own[fb] = g.g_loss[src];
        if (y < 0 || y >= g.V) own[fb] = NAN;
      }
      all[fb] = own[fb] + (g.g_lse ? g.g_lse[src] : 0.0f);
      const float lse = g.lse[src];
      if (lse != -INFINITY) {  // a class is left
        shift[fb] = lse;
        const int64_t in = y - f.first - static_cast<int64_t>(ia) * S::TA;
        if (in >= 0 && in < classes) want[fb] = static_cast<int>(in) - a0;
      }
    }
  }
  float* red = reinterpret_cast<float*>(lds);  // [WB][TA]
  // PLAIN: a whole tile without bias, where nothing is masked
  const auto gradients = [&](auto PLAIN) {
#pragma unroll
    for (int fa = 0; fa < S::FA; ++fa) {
      float bias[4], sum[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sum[r] = 0.0f;
        if (!PLAIN) bias[r] = a0 + fa * 16 + r < classes ? f.bias_of(at.a(fa) + r) : -INFINITY;
      }
#pragma unroll
      for (int fb = 0; fb < S::FB; ++fb) {
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (PLAIN) {
            d[r] = all[fb] * exp_of(acc[fa][fb][r] - shift[fb]);
          } else {
            d[r] = all[fb] * exp_of(acc[fa][fb][r] + bias[r] - shift[fb]);
            // rows behind the last, classes masked or behind the last: whatever they hold
            if (bias[r] == -INFINITY || shift[fb] == INFINITY) d[r] = 0.0f;
          }
        }
        if ((want[fb] >> 4) == fa) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((want[fb] & 15) == r) {
              d[r] -= own[fb];
              if (PARTS == 1) g.rest[at.b(fb)] = d[r] - __uint_as_float(rowvec::pack_bf16(d[r], 0.0f) << 16);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[fa][fb][r] = d[r];
          sum[r] += d[r];
        }
      }
      if (!PLAIN && g.bias_part) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sum[r] += xor_shfl<1>(sum[r]);
          sum[r] += xor_shfl<2>(sum[r]);
          sum[r] += xor_shfl<4>(sum[r]);
          sum[r] += xor_shfl<8>(sum[r]);
          if ((l & 15) == 0) red[(wave / S::WA) * S::TA + a0 + fa * 16 + r] = sum[r];
        }
      }
    }
  };
  if (!f.bias && rows == S::TB && classes == S::TA) {
    gradients(std::true_type());
  } else {
    gradients(std::false_type());
    if (g.bias_part) {
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < classes) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < S::WB; ++k) sum += red[k * S::TA + threadIdx.x];
        g.bias_part[static_cast<int64_t>(ib) * f.w.rows + static_cast<int64_t>(ia) * S::TA + threadIdx.x] = sum;
      }
      __syncthreads();
    }
  }
  if (!g.dz) return;
  // each part through LDS; zeros up to the next multiple of kStep of either axis
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
#pragma unroll
    for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
      for (int fb = 0; fb < S::FB; ++fb) {
        uint32_t lo[PARTS], hi[PARTS];
        split<PARTS>(acc[fa][fb][0], acc[fa][fb][1], lo);
        split<PARTS>(acc[fa][fb][2], acc[fa][fb][3], hi);
        stage<S>(lds, fa, fb, lo[q], hi[q]);
      }
    __syncthreads();
    store_tile<S, false>(lds, g.dz + q * g.part + static_cast<int64_t>(ib) * S::TB * g.ld + static_cast<int64_t>(ia) * S::TA,
                         g.ld, (rows + kStep - 1) / kStep * kStep, (classes + kStep - 1) / kStep * kStep);
    __syncthreads();
  }
}

// What is added to the weight's gradient for the labels' entries of the logits'
// gradient, the only large ones of their rows: what their rounding to bf16 left, to 8
// bits, times the rows (the gradient's error is then its own rounding, 1.7e-3, where it
// was that and the entries', 2.4e-3). x: the listed rows, x_width values of each.
struct Rests {
  const int32_t* mark;  // a listed row's label, or -1
  const float* rest;
  int64_t first;        // first class of the piece
  const uint16_t* x;
  int64_t ld;
};

// A workgroup's classes are b0 .. b0 + S::TB of the piece, its columns a0 ..: the rows
// whose label is among them are listed in their order (eight marks a thread at a
// time), their columns gathered into LDS, 64 rows at a time, and 32 are a product's
// step, the entries' rests one operand and the rows the other.
template <class S>
__device__ __forceinline__ void add_rests(const Rests& f, int64_t n, int64_t a0, int64_t b0, int64_t classes, char* lds,
                                          f32x4 (&acc)[S::FA][S::FB]) {
  constexpr int kWaves = S::kThreads / kWave, kEach = 8, kBatch = kEach * S::kThreads;
  constexpr int kList = kBatch + 4 * S::kThreads;  // entries
  constexpr int kGather = 64, kRow = S::TA * 2 + 16;
  int32_t* token = reinterpret_cast<int32_t*>(lds);
  int32_t* what = token + kList;  // its class in the tile
  float* rest = reinterpret_cast<float*>(what + kList);
  int32_t* votes = reinterpret_cast<int32_t*>(rest + kList);  // [kEach][kWaves]
  char* gathered = reinterpret_cast<char*>(votes + kEach * kWaves);
  static_assert(kList * 12 + kEach * kWaves * 4 + kGather * kRow <= S::kLdsBytes, "lists and rows in LDS");
  const int w = threadIdx.x / kWave, l = lane_id();
  const int col = (w % S::WA) * (S::TA / S::WA) + (l & 15), row = (w / S::WA) * (S::TB / S::WB) + (l & 15);
  int held = 0;
  for (int64_t r0 = 0; r0 < n; r0 += kBatch) {
    int in[kEach];
    uint64_t vote[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      in[i] = f.mark[min(r0 + i * S::kThreads + threadIdx.x, n - 1)] - static_cast<int>(f.first + b0);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      vote[i] = __ballot(r0 + i * S::kThreads + threadIdx.x < n && in[i] >= 0 && in[i] < classes);
      if (l == 0) votes[i * kWaves + w] = __popcll(vote[i]);
    }
    __syncthreads();
    int at = held;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      for (int k = 0; k < kWaves; ++k) {
        if (k == w && (vote[i] >> l & 1)) {
          const int64_t r = r0 + i * S::kThreads + threadIdx.x;
          const int to = at + __popcll(vote[i] & ((1ull << l) - 1));
          token[to] = static_cast<int32_t>(r);
          what[to] = in[i];
          rest[to] = f.rest[r];
        }
        at += votes[i * kWaves + k];
      }
    }
    held = at;
    __syncthreads();
    // on to the next marks while there is room for them
    if (held == 0 || (held <= kList - kBatch && r0 + kBatch < n)) continue;
    for (int i = held + threadIdx.x; i < (held + 31) / 32 * 32; i += S::kThreads) {
      token[i] = 0;
      what[i] = -1;
      rest[i] = 0.0f;
    }
    __syncthreads();
    for (int first = 0; first < held; first += kGather) {
      const int some = min(kGather, (held - first + 31) / 32 * 32);
      constexpr int kLanes = S::TA / 8;
#pragma unroll
      for (int j = 0; j < kGather * kLanes / S::kThreads; ++j) {
        const int i = j * S::kThreads + threadIdx.x, c = i % kLanes * 8;
        if (i / kLanes >= some) continue;
        U32x4 v{0, 0, 0, 0};
        if (a0 + c < f.ld) v = *reinterpret_cast<const U32x4*>(f.x + token[first + i / kLanes] * f.ld + a0 + c);
        *reinterpret_cast<U32x4*>(gathered + i / kLanes * kRow + c * 2) = v;
      }
      __syncthreads();
      for (int i = 0; i < some; i += 32) {
        const int k0 = i + (l >> 4) * 8;
        bf16x8 b[S::FB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int4 c = *reinterpret_cast<const int4*>(what + first + k0 + 4 * h);
          const float4 e = *reinterpret_cast<const float4*>(rest + first + k0 + 4 * h);
          const int cs[4] = {c.x, c.y, c.z, c.w};
          const float es[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int fb = 0; fb < S::FB; ++fb)
              b[fb][4 * h + k] = static_cast<__bf16>(cs[k] == row + fb * 16 ? es[k] : 0.0f);
        }
        // sixteen lanes' 8 bytes of four rows come back as four rows of one column a lane
        const char* from = gathered + (k0 + ((l & 15) >> 2)) * kRow + ((col & ~15) + (l & 3) * 4) * 2;
#pragma unroll
        for (int fa = 0; fa < S::FA; ++fa) {
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          typedef __attribute__((address_space(3))) s16x4* Turned;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Turned)(from + fa * 32));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Turned)(from + 4 * kRow + fa * 32));
          const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int fb = 0; fb < S::FB; ++fb)
            acc[fa][fb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[fb], acc[fa][fb], 0, 0, 0);
        }
      }
      __syncthreads();
    }
    held = 0;
  }
}

// out[b][a] = sum_k A[a][k] B[b][k], rows of out `ldo` values apart. SLOT: float32
// sums of a run of the K steps, blockIdx.y's, added to what earlier pieces left
// (accumulate); else rounded to T. The rows' gradient (ROWS): B's rows are those at
// work, A is the weight, turned; the weight's: they are the K axis, both are turned.
template <class S, typename T, int SEGS, bool SLOT, bool ROWS>
__global__ __launch_bounds__(S::kThreads, S::kGroups) void out_kernel(Operand a, Operand b, int ksteps,
                                                                  const int32_t* count, T* out, int64_t ldo,
                                                                  int64_t slot, int accumulate, Rests rests) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  if (ROWS) {
    b.rows = *count;
  } else {
    ksteps = (*count + kStep - 1) / kStep;
    a.depth = *count;
    b.depth = static_cast<int64_t>(ksteps) * kStep;
  }
  if (SLOT) {
    const int each = (ksteps + gridDim.y - 1) / gridDim.y, from = blockIdx.y * each;
    ksteps = max(0, min(each, ksteps - from));
    a.p += static_cast<int64_t>(from) * kStep * a.ld;
    a.depth -= static_cast<int64_t>(from) * kStep;
    b.p += static_cast<int64_t>(from) * kStep * (ROWS ? 1 : b.ld);
    b.depth -= static_cast<int64_t>(from) * kStep;
    out += blockIdx.y * slot;
  }
  const int ta = tiles(a.rows, S::TA), tb = tiles(b.rows, S::TB);
  if (static_cast<int64_t>(blockIdx.x) >= static_cast<int64_t>(ta) * tb) return;
  int ia, ib;
  ntgemm::tile_of(blockIdx.x, ta, tb, ia, ib);
  f32x4 acc[S::FA][S::FB];
  ntgemm::product<S, SEGS, true, !ROWS>(a, b, ia, ib, ksteps, lds, acc);
  if constexpr (SEGS == 1 && !ROWS)
    if (!SLOT || blockIdx.y == 0)
      add_rests<S>(rests, *count, static_cast<int64_t>(ia) * S::TA, static_cast<int64_t>(ib) * S::TB,
                   min(static_cast<int64_t>(S::TB), b.rows - static_cast<int64_t>(ib) * S::TB), lds, acc);
  const Place<S> at(ia, ib);
  if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
    for (int fb = 0; fb < S::FB; ++fb)
#pragma unroll
      for (int fa = 0; fa < S::FA; ++fa) {
        const f32x4 v = acc[fa][fb];
        stage<S>(lds, fa, fb, rowvec::pack_bf16(v[0], v[1]), rowvec::pack_bf16(v[2], v[3]));
      }
    __syncthreads();
    uint16_t* to = reinterpret_cast<uint16_t*>(out) + static_cast<int64_t>(ib) * S::TB * ldo + static_cast<int64_t>(ia) * S::TA;
    store_tile<S, true>(lds, to, ldo, static_cast<int>(min(static_cast<int64_t>(S::TB), b.rows - static_cast<int64_t>(ib) * S::TB)),
                     static_cast<int>(min(static_cast<int64_t>(S::TA), a.rows - static_cast<int64_t>(ia) * S::TA)));
  } else {
    typedef float Any __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int fb = 0; fb < S::FB; ++fb) {
      if (at.b(fb) >= b.rows) continue;
      T* row = out + at.b(fb) * ldo;
#pragma unroll
      for (int fa = 0; fa < S::FA; ++fa) {
        const int64_t i = at.a(fa);
        if (SLOT) {  // rows of a multiple of four floats
          f32x4* to = reinterpret_cast<f32x4*>(row + i);
          if (i < a.rows) *to = accumulate ? *to + acc[fa][fb] : acc[fa][fb];
        } else if (i + 4 <= a.rows) {
          *reinterpret_cast<Any*>(row + i) = acc[fa][fb];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (i + r < a.rows) row[i + r] = acc[fa][fb][r];
        }
      }
    }
  }
}

// Rows of a gradient from its slots' sums: grad_x of all rows from those of the rows
// with a gradient, by their places (zeros elsewhere), or without places.
template <typename T>
__global__ __launch_bounds__(kBlock) void rows_out_kernel(int64_t n, int D, const int32_t* place, const float* slots,
                                                          int ns, int64_t slot, int Dp, T* gx, const int32_t* mark,
                                                          const float* rest, const T* w, int64_t ldw, const void* bias,
                                                          int bias_f32) {
  const int64_t i = thread_of();
  const int per = Dp / 4;
  const int64_t r = i / per;
  const int c = static_cast<int>(i - r * per) * 4;
  if (r >= n) return;
  const int64_t p = place ? place[r] : r;
  f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
  if (p >= 0)
    for (int s = 0; s < ns; ++s) v += *reinterpret_cast<const f32x4*>(slots + s * slot + p * Dp + c);
  if (mark && p >= 0) {
    // what rounding left of the label's entry (Rests); a masked label's weight is not read
    const int y = mark[p];
    if (y >= 0 && !(bias && bias_at(bias, bias_f32, y) == -INFINITY)) {
      const T* row = w + y * ldw + c;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < D) v[k] = fmaf(rest[p], to_f32(row[k]), v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c + k < D) gx[r * D + c + k] = from_f32<T>(v[k]);
}

// grad_b of a piece from the sums of tiles of `tile` rows: 32 classes a workgroup, eight slices of the
// tiles, then the slices in order.
constexpr int kBiasCols = 32;
template <typename T>
__global__ __launch_bounds__(kBlock) void bias_kernel(const int32_t* count, int tile, int64_t V, const float* part, T* gb) {
  constexpr int kSlices = kBlock / kBiasCols;
  __shared__ float red[kSlices][kBiasCols];
  const int c = threadIdx.x % kBiasCols, k = threadIdx.x / kBiasCols;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kBiasCols + c;
  const int nt = tiles(*count, tile);
  float s = 0.0f;
  if (v < V)
    for (int t = k; t < nt; t += kSlices) s += part[t * V + v];
  red[k][c] = s;
  __syncthreads();
  if (k || v >= V) return;
#pragma unroll
  for (int t = 1; t < kSlices; ++t) s += red[t][c];
  gb[v] = from_f32<T>(s);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Rows that start 16-byte aligned.
bool rows_aligned(const void* p, int64_t ld, int64_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0;
}

// Rows that the tiles read where they lie (their offsets in a tile are 32 bits).
bool in_place(int dtype, int D, const void* p, int64_t ld) {
  return dtype == kBF16 && D % kStep == 0 && rows_aligned(p, ld, 2) && ld <= (1 << 24);
}

// Tiles of a product of A's and B's rows, with tiles of 256 or 128 rows.
int64_t tile_count(int64_t a, int64_t b, bool small) {
  const int64_t t = small ? Small::TA : Large::TA;
  return ((a + t - 1) / t) * ((b + t - 1) / t);
}

// Rounds of tiles over the card, in those of large ones: 256 at a time, or 512 small
// ones, two a CU, in 0.8 of that time for half of the products (up to 256 in 0.6;
// measured 0.76 to 0.89, and 0.55 to 0.61).
constexpr int kCus = 256;
double rounds(int64_t count, bool small) {
  if (!small) return static_cast<double>((count + kCus - 1) / kCus);
  return count <= kCus ? 0.6 : 0.8 * static_cast<double>((count + 2 * kCus - 1) / (2 * kCus));
}

// Whether the logits of a classes and b rows are formed in small tiles: where large
// ones leave CUs without work (412 rows against 10,093 classes of 3404 float32: 80
// large tiles 405 us, 316 small ones 308 us).
bool small_tiles(int64_t a, int64_t b) {
  return rounds(tile_count(a, b, true), true) < rounds(tile_count(a, b, false), false);
}

// A product whose K steps may be cut into slots.
struct Out {
  bool small;
  int splits;
};

// Few tiles: their K steps cut into slots, so that every CU has work, as long as a slot
// keeps eight steps; the tile by the rounds that takes, a slot's sums counted as two
// steps.
Out out_of(int64_t a, int64_t b, int64_t steps) {
  Out best{false, 1};
  double least = 0.0;
  for (int small = 0; small < 2; ++small) {
    const int64_t t = tile_count(a, b, small), room = small ? 2 * kCus : kCus;
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({room / std::max<int64_t>(1, t), steps / 8, 32}));
    const double time = rounds(t * splits, small) * static_cast<double>((steps + splits - 1) / splits) + 2.0 * splits;
    if (!small || time < least) {
      best = Out{small != 0, static_cast<int>(splits)};
      least = time;
    }
  }
  return best;
}

constexpr int kTile = Large::TA;  // pieces are a multiple of it

struct Cut {
  int parts, Kp;
  int64_t fwd_most;   // classes of a launch of the forward
  int64_t fwd_piece;  // classes packed at a time by it
  int64_t piece;      // classes of a piece of the backward
  int64_t rows_p;     // rows to the next multiple of kStep
  bool few, stream;   // the forward streams the classes, by stream_kernel,
  bool copied;        // which reads copies
  int tokens, groups, wide, few_grid, few_splits;
  bool stats_small, grad_small;
  Out dx, dw;         // the rows' gradient, in slots that the pieces add to; the weight's
  int Dp;
};

constexpr int64_t kPieceValues = 64ll << 20;   // of dz in a piece
constexpr int64_t kPackValues = 256ll << 20;   // of packed classes in a piece of the forward
constexpr int kFewSteps = 8;                   // of stream_kernel's run, at least
constexpr int64_t kMostTiles = 1 << 22;        // of a launch of the forward: 512 threads each, 32 bits of them

// Whether stream_kernel takes these.
bool streams(int dtype, int D, const void* x, int64_t ldx, const void* w, int64_t ldw) {
  const int64_t size = dtype == kF32 ? 4 : 2;
  return rows_aligned(x, ldx, size) && rows_aligned(w, ldw, size) && D * size % 128 == 0;
}

Cut cut(int dtype, int64_t n, int64_t V, int D, const void* x, int64_t ldx, const void* w, int64_t ldw) {
  Cut c;
  c.parts = dtype == kF32 ? 3 : 1;
  c.Kp = static_cast<int>(up(D, kStep));
  const auto even = [&](int64_t most) {
    most = std::max<int64_t>(kTile, most / kTile * kTile);
    const int64_t pieces = (V + most - 1) / most;
    return up((V + pieces - 1) / pieces, kTile);
  };
  c.fwd_most = kMostTiles / ((n + kTile - 1) / kTile + 1) * kTile;
  c.fwd_piece = even(std::min<int64_t>(kPackValues / (c.parts * static_cast<int64_t>(c.Kp)), c.fwd_most));
  c.rows_p = up(n, kStep);
  c.piece = even(std::min<int64_t>(kPieceValues / std::max<int64_t>(kStep, c.rows_p),
                                   kPackValues / (c.parts * static_cast<int64_t>(c.Kp))));
  c.Dp = static_cast<int>(up(D, 4));
  const int64_t most = std::min(c.piece, V);
  const int64_t some = std::min(c.fwd_piece, V);
  c.stats_small = small_tiles(some, n);
  const int64_t sets = (V + kFewClasses - 1) / kFewClasses, groups = (n + kFewRows - 1) / kFewRows;
  c.tokens = n <= 16 ? 16 : n <= 32 ? 32 : kFewRows;
  c.groups = static_cast<int>(groups);
  // Few wavefronts: runs of eight steps and more, where that gives a CU more of them, up
  // to four (1000 classes of 4096 float32: one row 93 -> 16 us, 64 rows 279 -> 40; two
  // runs gain nothing: 30,000 classes of 2048 bf16, one row, 25 -> 29).
  const int64_t steps = up(D, dtype == kF32 ? 32 : 64) / (dtype == kF32 ? 32 : 64), waves = sets * groups;
  const int64_t most_runs = std::min<int64_t>({4 * kCus / waves, steps / kFewSteps, 32});
  const int64_t each = most_runs > 2 ? (steps + most_runs - 1) / most_runs : std::max<int64_t>(1, steps);
  c.few_splits = static_cast<int>(std::max<int64_t>(1, (steps + each - 1) / each));
  // More rows of float32: by float32 products, 64 at a time, or packed for the tiles'
  // six of bf16. Microseconds of either, fitted to 131,072 x 4096 (128 rows 1.23 ms
  // streamed, 2.96 in tiles; 256 rows 2.31 and 3.30), 126,733 x 1184 (125 rows 0.38 and
  // 0.57; 192 rows 0.54 and 0.59), 1000 x 4096 (300 rows 60 us and 245), 10,000 x 512
  // (192 rows 48 and 58), 50,000 x 256 (192 rows 83 and 69), copied: 3000 x 4097 (200
  // rows 111 and 256), 50,001 x 1001 (100 rows 229 and 205).
  const double turns = waves <= 4 * kCus ? 1.0 : static_cast<double>(waves) / (4 * kCus) + 0.3;
  const double packs = 1.7e-6 * static_cast<double>(V + n) * D;  // or copies, where rows do not fill steps
  const double streamed = turns * (0.0754 * D / c.few_splits + 8.0) + (c.few_splits > 1 ? 10.0 : 0.0) +
                          (D % 32 ? packs : 0.0);
  const double tiled = packs + 15.0 + (c.stats_small ? 0.10 : 0.13) * c.Kp *
                       static_cast<double>((V + some - 1) / some) * rounds(tile_count(some, n, c.stats_small), c.stats_small);
  // Rows that stream_kernel cannot read are copied for it (up to 1 GB of them), so that
  // which of the two it is, and with it the result, hangs on the sizes alone.
  const bool aligned = streams(dtype, D, x, ldx, w, ldw);
  const bool more = n > kFewRows && dtype == kF32 && streamed < tiled && (aligned || V * up(D, 32) <= kPackValues);
  c.few = n <= kFewRows || more;
  c.copied = more && !aligned;
  c.stream = aligned || more;
  if (!c.few || !c.stream) c.few_splits = 1;
  c.wide = sets >= 64 ? 8 : 1;
  c.few_grid = c.few ? static_cast<int>(up(sets, c.wide) * groups) : 0;
  c.grad_small = small_tiles(most, n);
  c.dx = out_of(D, n, up(most, kStep) / kStep);
  c.dw = out_of(D, most, c.rows_p / kStep);
  return c;
}

// Bytes of a workspace's regions, 256-byte aligned.
struct Regions {
  int64_t total = 0;
  char* base;
  explicit Regions(void* p) : base(static_cast<char*>(p)) {}
  template <typename T>
  T* take(int64_t values) {
    T* p = base ? reinterpret_cast<T*>(base + total) : nullptr;
    total += up(values * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};

// Sets of classes whose statistics are joined.
int64_t stat_tiles(const Cut& c, int64_t n, int64_t V) {
  const int64_t classes = c.few ? kFewClasses : c.stats_small ? Small::TA : Large::TA;
  return (V + classes - 1) / classes;
}

struct FwdSpace {
  float2* part;
  float* chosen;
  f32x4* slots;
  float *copied_x, *copied_w;
  uint16_t *x, *w;
};

// x_in, w_in: read in place
int64_t fwd_space(const Cut& c, int64_t n, int64_t V, int D, bool x_in, bool w_in, void* p, FwdSpace* s) {
  Regions r(p);
  FwdSpace f;
  f.part = r.take<float2>(n * stat_tiles(c, n, V));
  f.chosen = r.take<float>(n);
  f.x = f.w = nullptr;
  f.slots = c.few_splits > 1 ? r.take<f32x4>(static_cast<int64_t>(c.few_splits) * c.few_grid * (c.tokens / 4) * kWave) : nullptr;
  f.copied_x = c.copied ? r.take<float>(n * up(D, 32)) : nullptr;
  f.copied_w = c.copied ? r.take<float>(V * up(D, 32)) : nullptr;
  if (!c.few) {
    if (!x_in) f.x = r.take<uint16_t>(c.parts * n * c.Kp);
    if (!w_in) f.w = r.take<uint16_t>(c.parts * std::min(c.fwd_piece, V) * c.Kp);
  }
  if (s) *s = f;
  return r.total;
}

struct BwdSpace {
  int32_t *list, *place, *count, *mark;
  float* rest;
  uint16_t *x, *w, *dz;
  float *slots, *wslots, *bias;
};

int64_t bwd_space(const Cut& c, int64_t n, int64_t V, bool w_in, int of, void* p, BwdSpace* s) {
  Regions r(p);
  BwdSpace b{};
  const int64_t vc = std::min(c.piece, up(V, kStep));
  b.list = r.take<int32_t>(n);
  b.place = r.take<int32_t>(n);
  b.count = r.take<int32_t>(1);
  b.mark = r.take<int32_t>(n);
  b.rest = r.take<float>(n);
  b.x = r.take<uint16_t>(c.parts * n * c.Kp);
  if (!w_in) b.w = r.take<uint16_t>(c.parts * vc * c.Kp);
  if (of & 3) b.dz = r.take<uint16_t>(c.parts * c.rows_p * vc);
  if (of & 1) b.slots = r.take<float>(c.dx.splits * n * c.Dp);
  if ((of & 2) && c.dw.splits > 1) b.wslots = r.take<float>(c.dw.splits * vc * c.Dp);
  if (of & 4) b.bias = r.take<float>(((n + Small::TB - 1) / Small::TB) * vc);
  if (s) *s = b;
  return r.total;
}

int check_args(const char* who, int dtype, int64_t n, int64_t V, int64_t D) {
  if (dtype != kF32 && dtype != kBF16) return set_error(kInvalid, "%s: dtype is 0 or 1", who);
  if (n < 0) return set_error(kInvalid, "%s: negative row count", who);
  if (n > kMaxRows) return set_error(kInvalid, "%s: more than %d rows", who, kMaxRows);
  if (V < 1 || V > kMaxClasses) return set_error(kInvalid, "%s: requires 1<=V<=%d", who, kMaxClasses);
  if (D < 1 || D > kMaxWidth) return set_error(kInvalid, "%s: requires 1<=D<=%d", who, kMaxWidth);
  return kOk;
}

// Workgroups for so many threads (thread_of), at most 2^23 along x: a launch's threads
// along an axis are 32 bits.
dim3 grid_of(int64_t threads) {
  const int64_t groups = (threads + kBlock - 1) / kBlock, x = std::min<int64_t>(groups, 1 << 23);
  return dim3(static_cast<uint32_t>(x), static_cast<uint32_t>((groups + x - 1) / x));
}

template <typename T, int PARTS>
int pack(hipStream_t st, int64_t n, const int32_t* count, const int32_t* list, int D, const T* src, int64_t ld,
         const void* bias, int bias_f32, uint16_t* dst, int Kp, int64_t part) {
  hipLaunchKernelGGL((pack_kernel<T, PARTS>), grid_of(n * (Kp / 8)), dim3(kBlock), 0, st, n, count, list, D, src, ld,
                     bias, bias_f32, dst, Kp, part);
  return check_launch("cign_linear_xent (pack)");
}

const void* bias_of(const void* bias, int f32, int64_t v) {
  return bias ? static_cast<const char*>(bias) + v * (f32 ? 4 : 2) : nullptr;
}

// f(Large()) or f(Small()), and the grid of its tiles.
template <class F>
void with_tiles(bool small, int64_t a, int64_t b, int splits, F&& f) {
  const dim3 grid(static_cast<uint32_t>(tile_count(a, b, small)), splits);
  if (small) f(Small(), grid);
  else f(Large(), grid);
}

template <typename T>
int forward(hipStream_t st, int64_t n, int V, int D, const T* x, int64_t ldx, const T* w, int64_t ldw, const void* bias,
            int bias_f32, const int64_t* labels, int64_t ignore, float* loss, float* lse, void* ws) {
  constexpr int dtype = std::is_same_v<T, float> ? kF32 : kBF16;
  constexpr int PARTS = dtype == kF32 ? 3 : 1, SEGS = PARTS == 3 ? 6 : 1;
  const Cut c = cut(dtype, n, V, D, x, ldx, w, ldw);
  const bool xin = in_place(dtype, D, x, ldx), win = in_place(dtype, D, w, ldw);
  FwdSpace s;
  fwd_space(c, n, V, D, xin, win, ws, &s);
  const int nt = static_cast<int>(stat_tiles(c, n, V));
  if (c.few) {
    if constexpr (std::is_same_v<T, float>)
      if (c.copied) {
        const int wide = static_cast<int>(up(D, 32));
        hipLaunchKernelGGL(copy_kernel, grid_of(n * (wide / 4)), dim3(kBlock), 0, st, n, D, x, ldx, s.copied_x, wide);
        hipLaunchKernelGGL(copy_kernel, grid_of(int64_t{V} * (wide / 4)), dim3(kBlock), 0, st, int64_t{V}, D, w, ldw,
                           s.copied_w, wide);
        x = s.copied_x;
        w = s.copied_w;
        ldx = ldw = D = wide;
      }
    const auto launch = [&](auto TC) {
      constexpr int TOKENS = decltype(TC)::value;
      if (c.stream)
        hipLaunchKernelGGL((stream_kernel<T, TOKENS>), dim3(c.few_grid, c.few_splits), dim3(kWave), 0, st, n, V, D, x,
                           ldx, w, ldw, bias, bias_f32, labels, s.part, s.chosen, c.groups, c.wide, s.slots);
      else
        hipLaunchKernelGGL((few_kernel<T, TOKENS>), dim3((nt + kWavesPerBlock - 1) / kWavesPerBlock), dim3(kBlock), 0, st,
                           n, V, D, x, ldx, w, ldw, bias, bias_f32, labels, s.part, s.chosen);
      if (s.slots)
        hipLaunchKernelGGL((few_join_kernel<TOKENS>), dim3(c.few_grid), dim3(kWave), 0, st, n, V, bias, bias_f32, labels,
                           s.part, s.chosen, c.groups, c.wide, s.slots, c.few_splits);
    };
    if (c.tokens == 16) launch(IC<16>());
    else if (c.tokens == 32) launch(IC<32>());
    else launch(IC<64>());
    if (const int rc = check_launch("cign_linear_xent_fwd")) return rc;
  } else {
    Operand xo{reinterpret_cast<const uint16_t*>(x), n, ldx, 0};
    if (!xin) {
      xo = Operand{s.x, n, c.Kp, n * c.Kp};
      if (const int rc = pack<T, PARTS>(st, n, nullptr, nullptr, D, x, ldx, nullptr, 0, s.x, c.Kp, xo.part)) return rc;
    }
    const int64_t piece = win ? c.fwd_most : c.fwd_piece;
    for (int64_t v = 0; v < V; v += piece) {
      const int64_t vn = std::min<int64_t>(piece, V - v);
      Operand wo{reinterpret_cast<const uint16_t*>(w + v * ldw), vn, ldw, 0};
      if (!win) {
        wo = Operand{s.w, vn, c.Kp, vn * c.Kp};
        if (const int rc = pack<T, PARTS>(st, vn, nullptr, nullptr, D, w + v * ldw, ldw, nullptr, 0, s.w, c.Kp, wo.part))
          return rc;
      }
      const Logits f{wo, xo, c.Kp / kStep, bias, bias_f32, v, nullptr, labels};
      with_tiles(c.stats_small, vn, n, 1, [&](auto shape, dim3 grid) {
        using S = decltype(shape);
        hipLaunchKernelGGL((stats_kernel<S, SEGS>), grid, dim3(S::kThreads), 0, st, f, n, s.part,
                           static_cast<int>(v / S::TA), s.chosen);
      });
      if (const int rc = check_launch("cign_linear_xent_fwd")) return rc;
    }
  }
  // a workgroup a row where there are few rows, 8 rows (64 bytes of a tile's) otherwise
  const auto joined = [&](auto RC) {
    constexpr int ROWS = decltype(RC)::value;
    hipLaunchKernelGGL((join_kernel<ROWS>), dim3(static_cast<uint32_t>((n + ROWS - 1) / ROWS)), dim3(kBlock), 0, st, n, V,
                       nt, s.part, labels, ignore, s.chosen, loss, lse);
  };
  if (c.few && n <= 512) joined(IC<1>());
  else joined(IC<8>());
  return check_launch("cign_linear_xent_fwd");
}

template <typename T>
int backward(hipStream_t st, int64_t n, int V, int D, const T* x, int64_t ldx, const T* w, int64_t ldw,
             const void* bias, int bias_f32, const int64_t* labels, int64_t ignore, const float* lse, const float* g_loss,
             const float* g_lse, T* gx, T* gw, void* gb, void* ws) {
  constexpr int dtype = std::is_same_v<T, float> ? kF32 : kBF16;
  constexpr int PARTS = dtype == kF32 ? 3 : 1, SEGS = PARTS == 3 ? 6 : 1;
  const char* who = "cign_linear_xent_bwd";
  const Cut c = cut(dtype, n, V, D, x, ldx, w, ldw);
  const int of = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0);
  const bool win = in_place(dtype, D, w, ldw) && !(bias && gx);  // masked classes are packed as zeros
  BwdSpace s;
  bwd_space(c, n, V, win, of, ws, &s);
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, st, n, labels, ignore, g_loss, g_lse,
                     static_cast<int64_t>(V), s.list, s.place, s.count, s.mark, s.rest);
  if (const int rc = check_launch(who)) return rc;
  const Operand xo{s.x, n, c.Kp, n * c.Kp};
  if (const int rc = pack<T, PARTS>(st, n, s.count, s.list, D, x, ldx, nullptr, 0, s.x, c.Kp, xo.part)) return rc;
  const Operand xt{s.x, D, c.Kp, n * c.Kp, c.Kp, 0};
  for (int64_t v = 0; v < V; v += c.piece) {
    const int64_t vn = std::min<int64_t>(c.piece, V - v), vp = up(vn, kStep);
    const T* wv = w + v * ldw;
    Operand wo{reinterpret_cast<const uint16_t*>(wv), vn, ldw, 0};
    if (!win) {
      wo = Operand{s.w, vn, c.Kp, vn * c.Kp};
      if (const int rc = pack<T, PARTS>(st, vn, nullptr, nullptr, D, wv, ldw, bias_of(bias, bias_f32, v), bias_f32, s.w,
                                            c.Kp, wo.part))
        return rc;
    }
    const Logits f{wo, xo, c.Kp / kStep, bias, bias_f32, v, s.count, labels};
    const int64_t dz_part = c.rows_p * vp;
    const Grads g{s.list, lse, g_loss, g_lse, ignore, V, s.dz, vp, dz_part, s.bias, s.rest};
    with_tiles(c.grad_small, vn, n, 1, [&](auto shape, dim3 grid) {
      using S = decltype(shape);
      hipLaunchKernelGGL((grad_kernel<S, SEGS>), grid, dim3(S::kThreads), 0, st, f, g);
    });
    if (const int rc = check_launch(who)) return rc;
    if (gx) {
      const Operand wt{wo.p, D, wo.ld, wo.part, c.Kp, vn};
      const Operand dz{s.dz, n, vp, dz_part};
      with_tiles(c.dx.small, D, n, c.dx.splits, [&](auto shape, dim3 grid) {
        using S = decltype(shape);
        hipLaunchKernelGGL((out_kernel<S, float, SEGS, true, true>), grid, dim3(S::kThreads), 0, st, wt, dz,
                           static_cast<int>(vp / kStep), s.count, s.slots, static_cast<int64_t>(c.Dp), n * c.Dp,
                           v > 0, Rests{});
      });
      if (const int rc = check_launch(who)) return rc;
    }
    if (gw) {
      const Operand dz{s.dz, vn, vp, dz_part, vp, 0};
      const Rests rests{PARTS == 1 ? s.mark : nullptr, s.rest, v, s.x, c.Kp};
      with_tiles(c.dw.small, D, vn, c.dw.splits, [&](auto shape, dim3 grid) {
        using S = decltype(shape);
        if (c.dw.splits > 1)
          hipLaunchKernelGGL((out_kernel<S, float, SEGS, true, false>), grid, dim3(S::kThreads), 0, st, xt, dz, 0, s.count,
                             s.wslots, static_cast<int64_t>(c.Dp), vn * c.Dp, 0, rests);
        else
          hipLaunchKernelGGL((out_kernel<S, T, SEGS, false, false>), grid, dim3(S::kThreads), 0, st, xt, dz, 0, s.count,
                             gw + v * D, static_cast<int64_t>(D), static_cast<int64_t>(0), 0, rests);
      });
      if (c.dw.splits > 1) {
        if (const int rc = check_launch(who)) return rc;
        hipLaunchKernelGGL((rows_out_kernel<T>), grid_of(vn * (c.Dp / 4)), dim3(kBlock), 0, st, vn, D,
                           static_cast<const int32_t*>(nullptr), s.wslots, c.dw.splits, vn * c.Dp, c.Dp, gw + v * D,
                           static_cast<const int32_t*>(nullptr), static_cast<const float*>(nullptr),
                           static_cast<const T*>(nullptr), static_cast<int64_t>(0), static_cast<const void*>(nullptr), 0);
      }
      if (const int rc = check_launch(who)) return rc;
    }
    if (gb) {
      const dim3 bias_grid(static_cast<uint32_t>((vn + kBiasCols - 1) / kBiasCols));
      if (bias_f32)
        hipLaunchKernelGGL((bias_kernel<float>), bias_grid, dim3(kBlock), 0, st, s.count, c.grad_small ? Small::TB : Large::TB, vn,
                           s.bias,
                           static_cast<float*>(gb) + v);
      else
        hipLaunchKernelGGL((bias_kernel<bf16>), bias_grid, dim3(kBlock), 0, st, s.count, c.grad_small ? Small::TB : Large::TB, vn,
                           s.bias,
                           static_cast<bf16*>(gb) + v);
      if (const int rc = check_launch(who)) return rc;
    }
  }
  if (gx) {
    hipLaunchKernelGGL((rows_out_kernel<T>), grid_of(n * (c.Dp / 4)), dim3(kBlock), 0, st, n, D, s.place, s.slots,
                       c.dx.splits, n * c.Dp, c.Dp, gx, PARTS == 1 ? s.mark : nullptr, s.rest, w, ldw, bias, bias_f32);
    return check_launch(who);
  }
  return kOk;
}

}  // namespace xent
}  // namespace cign

using namespace cign;
using namespace cign::xent;

extern "C" {

int64_t cign_linear_xent_workspace_bytes(int32_t dtype, int64_t n, int32_t V, int32_t D, const void* x,
                                         int64_t x_stride, const void* weight, int64_t weight_stride, int32_t of) {
  if (check_args("cign_linear_xent_workspace_bytes", dtype, n, V, D) || of < 0 || of > 7 || n == 0) return 0;
  const Cut c = cut(dtype, n, V, D, x, x_stride, weight, weight_stride);
  const bool xin = in_place(dtype, D, x, x_stride), win = in_place(dtype, D, weight, weight_stride);
  return of ? bwd_space(c, n, V, win && !(of & 1), of, nullptr, nullptr) : fwd_space(c, n, V, D, xin, win, nullptr, nullptr);
}

int cign_linear_xent_fwd(void* stream, int32_t dtype, int64_t n, int32_t V, int32_t D, const void* x, int64_t x_stride,
                         const void* weight, int64_t weight_stride, const void* bias, int32_t bias_dtype,
                         const int64_t* labels, int64_t ignore_index, float* loss, float* logsumexp, void* workspace,
                         int64_t workspace_bytes) {
  const char* who = "cign_linear_xent_fwd";
  if (const int rc = check_args(who, dtype, n, V, D)) return rc;
  if (bias && bias_dtype != kF32 && bias_dtype != dtype) return set_error(kInvalid, "%s: bias dtype", who);
  if (n == 0) return kOk;
  if (!x || !weight || !logsumexp || (loss == nullptr) != (labels == nullptr))
    return set_error(kInvalid, "%s: null argument", who);
  if (x_stride < 0 || weight_stride < 0) return set_error(kInvalid, "%s: negative row stride", who);
  if (!workspace ||
      workspace_bytes <
          cign_linear_xent_workspace_bytes(dtype, n, V, D, x, x_stride, weight, weight_stride, 0))
    return set_error(kInvalid, "%s: workspace too small", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kF32)
    return forward<float>(st, n, V, D, static_cast<const float*>(x), x_stride, static_cast<const float*>(weight),
                          weight_stride, bias, bias_dtype == kF32, labels, ignore_index, loss, logsumexp, workspace);
  return forward<bf16>(st, n, V, D, static_cast<const bf16*>(x), x_stride, static_cast<const bf16*>(weight),
                       weight_stride, bias, bias_dtype == kF32, labels, ignore_index, loss, logsumexp, workspace);
}

int cign_linear_xent_bwd(void* stream, int32_t dtype, int64_t n, int32_t V, int32_t D, const void* x, int64_t x_stride,
                         const void* weight, int64_t weight_stride, const void* bias, int32_t bias_dtype,
                         const int64_t* labels, int64_t ignore_index, const float* logsumexp, const float* grad_loss,
                         const float* grad_logsumexp, void* grad_x, void* grad_weight, void* grad_bias,
                         void* workspace, int64_t workspace_bytes) {
  const char* who = "cign_linear_xent_bwd";
  if (const int rc = check_args(who, dtype, n, V, D)) return rc;
  if ((bias || grad_bias) && bias_dtype != kF32 && bias_dtype != dtype)
    return set_error(kInvalid, "%s: bias dtype", who);
  const int of = (grad_x ? 1 : 0) | (grad_weight ? 2 : 0) | (grad_bias ? 4 : 0);
  if (!of) return kOk;
  if (n == 0) return set_error(kInvalid, "%s: no rows", who);
  if (!x || !weight || !logsumexp || (!grad_loss && !grad_logsumexp) || (grad_loss && !labels))
    return set_error(kInvalid, "%s: null argument", who);
  if (x_stride < 0 || weight_stride < 0) return set_error(kInvalid, "%s: negative row stride", who);
  if (!workspace ||
      workspace_bytes <
          cign_linear_xent_workspace_bytes(dtype, n, V, D, x, x_stride, weight, weight_stride, of))
    return set_error(kInvalid, "%s: workspace too small", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kF32)
    return backward<float>(st, n, V, D, static_cast<const float*>(x), x_stride, static_cast<const float*>(weight),
                           weight_stride, bias, bias_dtype == kF32, labels, ignore_index, logsumexp, grad_loss,
                           grad_logsumexp, static_cast<float*>(grad_x), static_cast<float*>(grad_weight), grad_bias,
                           workspace);
  return backward<bf16>(st, n, V, D, static_cast<const bf16*>(x), x_stride, static_cast<const bf16*>(weight),
                        weight_stride, bias, bias_dtype == kF32, labels, ignore_index, logsumexp, grad_loss,
                        grad_logsumexp, static_cast<bf16*>(grad_x), static_cast<bf16*>(grad_weight), grad_bias,
                        workspace);
}

}  // extern "C"

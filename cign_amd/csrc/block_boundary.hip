// The boundary of two blocks, rows of 1 <= D <= 8192 values, float32 or bf16: the
// norm of a block's branch u, its gate a and residual scale c, the residual h and
// the next block's norm,
//   v = N(u) w1 + b1, s = sigmoid(a), hidden = h + c s v, y = N(hidden) w2 + b2,
// N a LayerNorm ((t - mean) rstd) or an RMS norm (t rstd). Backward, with g1 and g2
// the gradients of hidden and y, n = N(hidden), m = N(u), d2 = g2 w2:
//   gh = g1 + rstd2 (d2 - mean(d2) - n mean(d2 n))        (RMS: no mean(d2))
//   gv = gh c s, d1 = gv w1, grad_u = rstd1 (d1 - mean(d1) - m mean(d1 m)),
//   grad_h = gh, grad_a = gh c v s (1 - s), its sum where a row has one gate,
//   grad_w1 = sum gv m, grad_b1 = sum gv, grad_c = sum gh s v, grad_w2 = sum g2 n,
//   grad_b2 = sum g2.
//
// Both passes are streams, as the LayerNorm's (layernorm.hip): each array is read
// once and written once, a row stays in the registers of NT threads, and what the
// vectors' gradients take is added up per thread over a workgroup's rows, one
// partial row a workgroup, which param_kernel adds in a fixed order. hidden is
// normed as float32, before it is rounded to the rows' type; the backward forms it
// again from u, h and a, so that both see the same values.
//
// HBM bounds the large ones (a copy of 4 GiB moves 4.75 TB/s), latency and two waves
// of workgroups the small. Measured, forward / backward / vectors:
//   16,384 x 4096 bf16, a gate a value   125 us (5.4 TB/s) / 195 (5.5) / 5
//   24,492 x 256 f32, a gate a row        17 us (5.9) / 30 (5.0) / 4
//   10,007 x 1001 bf16, a gate a value    23 us (4.3) / 43 (3.7) / 5
//   8192 x 8192 bf16                     157 us (4.3) / 326 (3.3); with 1024 threads, whose
//     128 registers do not hold the backward's values, 172 / 777
//   one row of 4096                      2.8 us, a launch and two reductions
#include "rowops.h"
#include "rowvec.h"

namespace cign {
namespace boundary {
using namespace rowvec;

constexpr int kMaxWidth = 8192;
constexpr int kVectors = 5;      // w1, b1, c, w2, b2
constexpr int kMostKept = 8;     // values of a row's array in a thread with which the vectors stay in registers too

enum Gate : int { kNoGate = 0, kRowGate = 1, kValueGate = 2 };

template <int N>
using IC = std::integral_constant<int, N>;

template <int NT>
struct Shape {
  static constexpr int kThreads = NT <= kWave ? kBlock : NT;
  static constexpr int kRows = kThreads / NT;
  static constexpr int kSlots = NT > kWave ? 2 * (NT / kWave) : 1;
};

struct Args {
  int64_t n;
  int D;
  const void *branch, *residual, *gate;
  int64_t ldu, ldh, lda;
  const void* vec[kVectors];  // w1, b1, c, w2, b2 or null (ones, zeros, ones, ones, zeros)
  float eps;
  // forward
  void *hidden, *y;
  float* stats;  // [4][n]: mean and rstd of the branch, of hidden; or null
  // backward
  const void *g1, *g2;  // or null
  int64_t ld1, ld2;
  void *gu, *gh, *ga;   // or null
  float* part;          // [kVectors][nb][D] or null
  int nb;
};

__device__ __forceinline__ float sigmoid(float a) {
  // 1 / (1 + e^-a), both exact to 2 ulp; e^-a is inf for a < -88, and s then 0
  return 1.0f / (1.0f + __expf(-a));
}

template <typename T, int W, bool PAST>
__device__ __forceinline__ void store_own(T* row, int at, int own, const float (&v)[W]) {
  if (own == 0) {
    if constexpr (PAST)
      RowChunk<T, W>::store_past(row + at, v);
    else
      RowChunk<T, W>::store(row + at, v);
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w >= own) row[at + w] = from_f32<T>(v[w]);
  }
}

// Chunks of the five vectors: kept as they are stored, or (WIDE, where a thread's
// registers hold 16 values of each array of a row) read from the cache at each use.
template <typename TW, int W, int V, bool WIDE>
struct Vectors {
  using P = RowChunk<TW, W>;
  typename P::Raw raw[WIDE ? 1 : kVectors][WIDE ? 1 : V];
  const TW* from[kVectors];
  int at[V];
  __device__ __forceinline__ Vectors(const Args& k, const int (&place)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) at[v] = place[v];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      from[i] = static_cast<const TW*>(k.vec[i]);
      if constexpr (!WIDE)
        if (from[i])
#pragma unroll
          for (int v = 0; v < V; ++v) raw[i][v] = P::load(from[i] + at[v]);
    }
  }
  __device__ __forceinline__ void get(int i, int v, float none, float (&out)[W]) const {
    if (from[i]) {
      if constexpr (WIDE) P::unpack(P::load(from[i] + at[v]), out);
      else P::unpack(raw[i][v], out);
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) out[w] = none;
    }
  }
};

// What a thread adds up over its rows for the vectors' gradients: in registers, or
// (WIDE) all but the last vector's in LDS, 128 KB, 16 bytes a thread next to each other.
template <int W, int V, int NT, bool WIDE>
struct Sums {
  float acc[WIDE ? 1 : kVectors][V][W];
  float* lds;  // [4][V * W / 4][NT][4]
  __device__ __forceinline__ explicit Sums(float* where) : lds(where + threadIdx.x * 4) {
    if constexpr (WIDE)
      for (int j = 0; j < 4 * V * W / 4; ++j) *reinterpret_cast<float4*>(lds + j * NT * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < (WIDE ? 1 : kVectors); ++i)
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int w = 0; w < W; ++w) acc[i][v][w] = 0.0f;
  }
  __device__ __forceinline__ float4* at(int i, int v, int j) const {
    return reinterpret_cast<float4*>(lds + ((i * V + v) * (W / 4) + j) * NT * 4);
  }
  __device__ __forceinline__ void add(int i, int v, const float (&t)[W]) {
    if (!WIDE || i == 4) {
#pragma unroll
      for (int w = 0; w < W; ++w) acc[WIDE ? 0 : i][v][w] += t[w];
    } else {
      if constexpr (WIDE)
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
          float4 s = *at(i, v, j);
          s.x += t[4 * j];
          s.y += t[4 * j + 1];
          s.z += t[4 * j + 2];
          s.w += t[4 * j + 3];
          *at(i, v, j) = s;
        }
    }
  }
  __device__ __forceinline__ void get(int i, int v, float (&t)[W]) const {
    if (!WIDE || i == 4) {
#pragma unroll
      for (int w = 0; w < W; ++w) t[w] = acc[WIDE ? 0 : i][v][w];
    } else {
      if constexpr (WIDE)
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
          const float4 s = *at(i, v, j);
          t[4 * j] = s.x;
          t[4 * j + 1] = s.y;
          t[4 * j + 2] = s.z;
          t[4 * j + 3] = s.w;
        }
    }
  }
};

// mean and rstd of a row's values, in place: t becomes the centred values (LAYER).
template <bool LAYER, int W, int V, int NT>
__device__ __forceinline__ void moments(GroupReduce<NT, 1>& reduce, float (&t)[V][W], const int (&own)[V], float inv,
                                        float eps, float& mean, float& rstd) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (LAYER) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int w = 0; w < W; ++w) s[0] += w >= own[v] ? t[v][w] : 0.0f;
    reduce.sum(s);
    mean = s[0] * inv;
    s[0] = 0.0f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (LAYER) t[v][w] -= mean;
      s[0] += w >= own[v] ? t[v][w] * t[v][w] : 0.0f;
    }
  reduce.sum(s);
  rstd = 1.0f / sqrtf(s[0] * inv + eps);
}

template <typename T, typename TW, int W, int NT, int V, int GATE, bool LAYER, bool PAST>
__global__ __launch_bounds__(Shape<NT>::kThreads) void fwd_kernel(Args k) {
  using X = RowChunk<T, W>;
  __shared__ float slots[Shape<NT>::kSlots][1];
  GroupReduce<NT, 1> reduce(slots);
  const int q = threadIdx.x & (NT - 1);
  const T *branch = static_cast<const T*>(k.branch), *residual = static_cast<const T*>(k.residual),
          *gate = static_cast<const T*>(k.gate);
  int at[V], own[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = q + v * NT;
    at[v] = chunk_start<W>(c, k.D);
    own[v] = c * W - at[v];
  }
  const Vectors<TW, W, V, (V * W > kMostKept)> p(k, at);
  const float inv = 1.0f / static_cast<float>(k.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * Shape<NT>::kRows;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * Shape<NT>::kRows + threadIdx.x / NT; r < k.n; r += step) {
    typename X::Raw ur[V], hr[V], ar[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ur[v] = X::load(branch + r * k.ldu + at[v]);
      hr[v] = X::load(residual + r * k.ldh + at[v]);
      if (GATE == kValueGate) ar[v] = X::load(gate + r * k.lda + at[v]);
    }
    const float open = GATE == kRowGate ? sigmoid(to_f32(gate[r * k.lda])) : 1.0f;
    float t[V][W], mean1, rstd1, mean2, rstd2;
#pragma unroll
    for (int v = 0; v < V; ++v) X::unpack(ur[v], t[v]);
    moments<LAYER>(reduce, t, own, inv, k.eps, mean1, rstd1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float h[W], a[W], w1[W], b1[W], c[W];
      X::unpack(hr[v], h);
      if (GATE == kValueGate) X::unpack(ar[v], a);
      p.get(0, v, 1.0f, w1);
      p.get(1, v, 0.0f, b1);
      p.get(2, v, 1.0f, c);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float s = GATE == kValueGate ? sigmoid(a[w]) : open;
        t[v][w] = fmaf(c[w] * s, fmaf(t[v][w] * rstd1, w1[w], b1[w]), h[w]);
      }
      if (own[v] < W) store_own<T, W, PAST>(static_cast<T*>(k.hidden) + r * k.D, at[v], own[v], t[v]);
    }
    moments<LAYER>(reduce, t, own, inv, k.eps, mean2, rstd2);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w2[W], b2[W];
      p.get(3, v, 1.0f, w2);
      p.get(4, v, 0.0f, b2);
#pragma unroll
      for (int w = 0; w < W; ++w) t[v][w] = fmaf(t[v][w] * rstd2, w2[w], b2[w]);
      if (own[v] < W) store_own<T, W, PAST>(static_cast<T*>(k.y) + r * k.D, at[v], own[v], t[v]);
    }
    if (q == 0 && k.stats) {
      k.stats[r] = mean1;
      k.stats[k.n + r] = rstd1;
      k.stats[2 * k.n + r] = mean2;
      k.stats[3 * k.n + r] = rstd2;
    }
  }
}

template <typename T, typename TW, int W, int NT, int V, int GATE, bool LAYER, bool PAST>
__global__ __launch_bounds__(Shape<NT>::kThreads) void bwd_kernel(Args k) {
  using X = RowChunk<T, W>;
  constexpr int kRows = Shape<NT>::kRows;
  constexpr int kSums = 3;
  __shared__ float slots[Shape<NT>::kSlots][kSums];
  GroupReduce<NT, kSums> reduce(slots);
  const int q = threadIdx.x & (NT - 1), slot = threadIdx.x / NT;
  const T *branch = static_cast<const T*>(k.branch), *residual = static_cast<const T*>(k.residual),
          *gate = static_cast<const T*>(k.gate), *g1 = static_cast<const T*>(k.g1), *g2 = static_cast<const T*>(k.g2);
  int at[V], own[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = q + v * NT;
    at[v] = chunk_start<W>(c, k.D);
    own[v] = c * W - at[v];
  }
  constexpr bool kWide = V * W > kMostKept;
  constexpr int kCells = NT * V * W;
  __shared__ float lds[kWide ? 4 * kCells : kRows > 1 ? kRows * kCells : 1];
  const Vectors<TW, W, V, kWide> p(k, at);
  Sums<W, V, NT, kWide> sum(lds);
  const float inv = 1.0f / static_cast<float>(k.D);
  const int64_t step = static_cast<int64_t>(k.nb) * kRows;
  int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + slot;
  typename X::Raw un[V], hn[V], an[V], n1[V], nn2[V];
  float openn = 1.0f, kept[4];
  const auto load = [&](int64_t row) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      un[v] = X::load(branch + row * k.ldu + at[v]);
      hn[v] = X::load(residual + row * k.ldh + at[v]);
      if (GATE == kValueGate) an[v] = X::load(gate + row * k.lda + at[v]);
      if (g1) n1[v] = X::load(g1 + row * k.ld1 + at[v]);
      if (g2) nn2[v] = X::load(g2 + row * k.ld2 + at[v]);
    }
    if (GATE == kRowGate) openn = to_f32(gate[row * k.lda]);
#pragma unroll
    for (int i = 0; i < 4; ++i) kept[i] = k.stats[i * k.n + row];
  };
  // eight values a thread: the next row's loads go out before this row's sums (16,384 x
  // 4096 bf16 195 us, 242 without; four values 220, 213 without; 16 do not fit)
  constexpr bool kAhead = V * W == kMostKept;
  if (kAhead && r < k.n) load(r);
  for (; r < k.n; r += step) {
    if (!kAhead) load(r);
    typename X::Raw ur[V], hr[V], ar[V], r1[V], r2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ur[v] = un[v];
      hr[v] = hn[v];
      if (GATE == kValueGate) ar[v] = an[v];
      if (g1) r1[v] = n1[v];
      if (g2) r2[v] = nn2[v];
    }
    const float mean1 = kept[0], rstd1 = kept[1], mean2 = kept[2], rstd2 = kept[3];
    const float open = GATE == kRowGate ? sigmoid(openn) : 1.0f;
    if (kAhead) load(r + step < k.n ? r + step : r);
    float m[V][W], s[V][W], n2[V][W], g[V][W];
    float sums[kSums] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float h[W], w1[W], b1[W], c[W], w2[W], along[W];
      X::unpack(ur[v], m[v]);
      X::unpack(hr[v], h);
      if (GATE == kValueGate) X::unpack(ar[v], s[v]);
      if (g2) {
        X::unpack(r2[v], g[v]);
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w) g[v][w] = 0.0f;
      }
      p.get(0, v, 1.0f, w1);
      p.get(1, v, 0.0f, b1);
      p.get(2, v, 1.0f, c);
      p.get(3, v, 1.0f, w2);
      sum.add(4, v, g[v]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // the forward's operations, in its order
        const float centred = LAYER ? m[v][w] - mean1 : m[v][w];
        m[v][w] = centred * rstd1;
        s[v][w] = GATE == kValueGate ? sigmoid(s[v][w]) : open;
        const float hidden = fmaf(c[w] * s[v][w], fmaf(m[v][w], w1[w], b1[w]), h[w]);
        n2[v][w] = (LAYER ? hidden - mean2 : hidden) * rstd2;
        along[w] = g[v][w] * n2[v][w];
        g[v][w] *= w2[w];
        if (LAYER) sums[0] += w >= own[v] ? g[v][w] : 0.0f;
        sums[1] += w >= own[v] ? g[v][w] * n2[v][w] : 0.0f;
      }
      sum.add(3, v, along);
    }
    reduce.sum(sums);
    const float c1 = LAYER ? sums[0] * inv : 0.0f, c2 = sums[1] * inv;
    sums[0] = sums[1] = sums[2] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float first[W], w1[W], b1[W], c[W], ga[W], to_c[W], gv[W], to_w1[W];
      if (g1) {
        X::unpack(r1[v], first);
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w) first[w] = 0.0f;
      }
      p.get(0, v, 1.0f, w1);
      p.get(1, v, 0.0f, b1);
      p.get(2, v, 1.0f, c);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float gh = fmaf(rstd2, g[v][w] - c1 - n2[v][w] * c2, first[w]);
        g[v][w] = gh;
        const float val = fmaf(m[v][w], w1[w], b1[w]);
        const float open_v = s[v][w] * val;
        to_c[w] = gh * open_v;
        ga[w] = gh * c[w] * open_v * (1.0f - s[v][w]);
        if (GATE == kRowGate) sums[2] += w >= own[v] ? ga[w] : 0.0f;
        gv[w] = gh * c[w] * s[v][w];
        to_w1[w] = gv[w] * m[v][w];
        n2[v][w] = gv[w] * w1[w];  // d1
        if (LAYER) sums[0] += w >= own[v] ? n2[v][w] : 0.0f;
        sums[1] += w >= own[v] ? n2[v][w] * m[v][w] : 0.0f;
      }
      sum.add(2, v, to_c);
      sum.add(1, v, gv);
      sum.add(0, v, to_w1);
      if (own[v] < W) {
        if (k.gh) store_own<T, W, PAST>(static_cast<T*>(k.gh) + r * k.D, at[v], own[v], g[v]);
        if (GATE == kValueGate && k.ga) store_own<T, W, PAST>(static_cast<T*>(k.ga) + r * k.D, at[v], own[v], ga);
      }
    }
    if (k.gu || (GATE == kRowGate && k.ga)) {
      reduce.sum(sums);
      const float e1 = LAYER ? sums[0] * inv : 0.0f, e2 = sums[1] * inv;
      if (k.gu)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (own[v] >= W) continue;
          float o[W];
#pragma unroll
          for (int w = 0; w < W; ++w) o[w] = rstd1 * (n2[v][w] - e1 - m[v][w] * e2);
          store_own<T, W, PAST>(static_cast<T*>(k.gu) + r * k.D, at[v], own[v], o);
        }
      if (GATE == kRowGate && k.ga && q == 0) static_cast<T*>(k.ga)[r] = from_f32<T>(sums[2]);
    }
  }
  if (!k.part) return;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float t[W];
        sum.get(i, v, t);
        if (own[v] < W)
          store_own<float, W, false>(k.part + (static_cast<int64_t>(i) * k.nb + blockIdx.x) * k.D, at[v], own[v], t);
      }
  } else {
    // the workgroup's row slots, added in order
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float t[W];
        sum.get(i, v, t);
#pragma unroll
        for (int w = 0; w < W; ++w) lds[slot * kCells + (q + v * NT) * W + w] = t[w];
      }
      __syncthreads();
      float* dst = k.part + (static_cast<int64_t>(i) * k.nb + blockIdx.x) * k.D;
      for (int j = threadIdx.x; j < kCells; j += kBlock) {
        const int c = j / W;
        const int col = chunk_start<W>(c, k.D) + j % W;
        if (c * W >= k.D || col < c * W) continue;  // past the row, or another chunk's
        float total = 0.0f;
        for (int t = 0; t < kRows; ++t) total += lds[t * kCells + j];
        dst[col] = total;
      }
    }
  }
}

// The vectors' gradients from the nb partial rows of each, 32 columns a
// workgroup, 32 slices of the rows at a time, then the slices in an LDS tree.
constexpr int kParamCols = 32, kParamThreads = 1024;
struct Outs {
  void* p[kVectors];
};

template <typename TW>
__global__ __launch_bounds__(kParamThreads) void param_kernel(const float* part, int nb, int D, Outs outs) {
  constexpr int kSlices = kParamThreads / kParamCols;
  __shared__ float red[kParamThreads];
  TW* out = static_cast<TW*>(outs.p[blockIdx.y]);
  if (!out) return;
  const float* src = part + static_cast<int64_t>(blockIdx.y) * nb * D;
  const int c = blockIdx.x * kParamCols + threadIdx.x % kParamCols;
  const int s = threadIdx.x / kParamCols;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < D) {
    int b = s;
    for (; b + 3 * kSlices < nb; b += 4 * kSlices)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] += src[static_cast<int64_t>(b + u * kSlices) * D + c];
    for (; b < nb; b += kSlices) acc[0] += src[static_cast<int64_t>(b) * D + c];
  }
  red[threadIdx.x] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  for (int h = kSlices / 2; h > 0; h >>= 1) {
    if (s < h) red[threadIdx.x] += red[threadIdx.x + h * kParamCols];
    __syncthreads();
  }
  if (s == 0 && c < D) out[c] = from_f32<TW>(red[threadIdx.x]);
}

// f(IC<W>, IC<NT>, IC<V>): one chunk a thread, lanes of a wavefront or a workgroup of
// 128 to 512 threads (10,007 x 1001 bf16 backward by 128 threads 43 us, by 64 lanes of
// two chunks 59); beyond 4096 bf16 or 2048 float32 columns several chunks.
template <typename T, class F>
int with_shape(int D, F&& f) {
  constexpr int W = kChunk<T>;
  if (D < W) {
    if (D <= 1) return f(IC<1>(), IC<1>(), IC<1>());
    if (D <= 2) return f(IC<1>(), IC<2>(), IC<1>());
    if (D <= 4) return f(IC<1>(), IC<4>(), IC<1>());
    return f(IC<1>(), IC<8>(), IC<1>());
  }
  const int nc = (D + W - 1) / W;
  if (nc <= 4) return f(IC<W>(), IC<4>(), IC<1>());
  if (nc <= 16) return f(IC<W>(), IC<16>(), IC<1>());
  if (nc <= 32) return f(IC<W>(), IC<32>(), IC<1>());
  if (nc <= 64) return f(IC<W>(), IC<64>(), IC<1>());
  if (nc <= 128) return f(IC<W>(), IC<128>(), IC<1>());
  if (nc <= 256) return f(IC<W>(), IC<256>(), IC<1>());
  if (nc <= 512) return f(IC<W>(), IC<512>(), IC<1>());
  if (nc <= 1024) return f(IC<W>(), IC<512>(), IC<2>());
  if constexpr (W == 4) return f(IC<W>(), IC<512>(), IC<4>());
  return static_cast<int>(kInvalid);  // D <= 8192
}

template <class F>
int with_types(int x_dtype, int w_dtype, F&& f) {
  if (x_dtype == kF32) return f(float(), float());
  if (w_dtype == kF32) return f(bf16(), float());
  return f(bf16(), bf16());
}

template <class F>
int with_form(int gate, int layer, bool past, F&& f) {
  const auto g = [&](auto L, auto P) {
    if (gate == kNoGate) return f(IC<kNoGate>(), L, P);
    if (gate == kRowGate) return f(IC<kRowGate>(), L, P);
    return f(IC<kValueGate>(), L, P);
  };
  const auto l = [&](auto P) { return layer ? g(std::true_type(), P) : g(std::false_type(), P); };
  return past ? l(std::true_type()) : l(std::false_type());
}

// Arrays of this many bytes and more are written past the cache.
constexpr int64_t kPastBytes = 112ll << 20;

int check_args(const char* who, int64_t n, int D, int x_dtype, int w_dtype, int gate_kind, int layer) {
  if (n < 0) return set_error(kInvalid, "%s: negative row count", who);
  if (D < 1 || D > kMaxWidth) return set_error(kInvalid, "%s: requires 1<=D<=%d, got %d", who, kMaxWidth, D);
  if ((x_dtype != kF32 && x_dtype != kBF16) || (w_dtype != kF32 && w_dtype != x_dtype))
    return set_error(kInvalid, "%s: dtypes are 0 or 1, the vectors' 0 or the rows'", who);
  if (gate_kind < kNoGate || gate_kind > kValueGate) return set_error(kInvalid, "%s: gate is 0, 1 or 2", who);
  if (layer != 0 && layer != 1) return set_error(kInvalid, "%s: layer is 0 or 1", who);
  return kOk;
}

// Workgroups of the backward, its partial rows: what the card holds at a time.
int bwd_blocks(int64_t n, int rows, int threads) {
  const int64_t groups = (n + rows - 1) / rows, most = threads > kBlock ? 256 : rows > 1 ? 512 : 1024;
  return static_cast<int>(groups < most ? groups : most);
}

}  // namespace boundary
}  // namespace cign

using namespace cign;
using namespace cign::boundary;

extern "C" {

int cign_block_boundary_fwd(void* stream, int64_t n, int32_t D, int32_t x_dtype, int32_t w_dtype, int32_t layer,
                            int32_t gate_kind, const void* branch, int64_t branch_stride, const void* residual,
                            int64_t residual_stride, const void* gate, int64_t gate_stride, const void* post_weight,
                            const void* post_bias, const void* scale, const void* next_weight, const void* next_bias,
                            float eps, void* hidden, void* y, float* stats) {
  const char* who = "cign_block_boundary_fwd";
  if (const int rc = check_args(who, n, D, x_dtype, w_dtype, gate_kind, layer)) return rc;
  if (n == 0) return kOk;
  if (!branch || !residual || !hidden || !y || (gate_kind != kNoGate && !gate))
    return set_error(kInvalid, "%s: null argument", who);
  if (branch_stride < 0 || residual_stride < 0 || gate_stride < 0)
    return set_error(kInvalid, "%s: negative row stride", who);
  Args k{};
  k.n = n;
  k.D = D;
  k.branch = branch;
  k.residual = residual;
  k.gate = gate;
  k.ldu = branch_stride;
  k.ldh = residual_stride;
  k.lda = gate_stride;
  const void* vec[kVectors] = {post_weight, post_bias, scale, next_weight, next_bias};
  for (int i = 0; i < kVectors; ++i) k.vec[i] = vec[i];
  k.eps = eps;
  k.hidden = hidden;
  k.y = y;
  k.stats = stats;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using TW = decltype(tw);
    return with_shape<T>(D, [&](auto WC, auto NC, auto VC) {
      constexpr int W = decltype(WC)::value, NT = decltype(NC)::value, V = decltype(VC)::value;
      return with_form(gate_kind, layer, n * D * static_cast<int64_t>(sizeof(T)) >= kPastBytes, [&](auto GC, auto LC, auto PC) {
        const int64_t groups = (n + Shape<NT>::kRows - 1) / Shape<NT>::kRows;
        const int grid = static_cast<int>(groups < 2048 ? groups : 2048);
        hipLaunchKernelGGL((fwd_kernel<T, TW, W, NT, V, decltype(GC)::value, decltype(LC)::value,
                                        decltype(PC)::value>), dim3(grid),
                           dim3(Shape<NT>::kThreads), 0, st, k);
        return check_launch(who);
      });
    });
  });
}

int64_t cign_block_boundary_bwd_workspace_bytes(int64_t n, int32_t D) {
  if (n < 0 || D < 1 || D > kMaxWidth) return 0;
  return kVectors * static_cast<int64_t>(sizeof(float)) * bwd_blocks(n, 1, kBlock) * D;
}

int cign_block_boundary_bwd(void* stream, int64_t n, int32_t D, int32_t x_dtype, int32_t w_dtype, int32_t layer,
                            int32_t gate_kind, const void* grad_hidden, int64_t grad_hidden_stride, const void* grad_y,
                            int64_t grad_y_stride, const void* branch, int64_t branch_stride, const void* residual,
                            int64_t residual_stride, const void* gate, int64_t gate_stride, const void* post_weight,
                            const void* post_bias, const void* scale, const void* next_weight, const float* stats,
                            void* grad_branch, void* grad_residual, void* grad_gate, void* grad_post_weight,
                            void* grad_post_bias, void* grad_scale, void* grad_next_weight, void* grad_next_bias,
                            void* workspace, int64_t workspace_bytes) {
  const char* who = "cign_block_boundary_bwd";
  if (const int rc = check_args(who, n, D, x_dtype, w_dtype, gate_kind, layer)) return rc;
  const Outs outs{{grad_post_weight, grad_post_bias, grad_scale, grad_next_weight, grad_next_bias}};
  bool params = false;
  for (void* p : outs.p) params = params || p;
  if (!params && (n == 0 || (!grad_branch && !grad_residual && !grad_gate))) return kOk;
  if (n > 0 && (!branch || !residual || !stats || (gate_kind != kNoGate && !gate) || (!grad_hidden && !grad_y)))
    return set_error(kInvalid, "%s: null argument", who);
  if (branch_stride < 0 || residual_stride < 0 || gate_stride < 0 || grad_hidden_stride < 0 || grad_y_stride < 0)
    return set_error(kInvalid, "%s: negative row stride", who);
  if (params && n > 0 && (!workspace || workspace_bytes < cign_block_boundary_bwd_workspace_bytes(n, D)))
    return set_error(kInvalid, "%s: workspace too small", who);
  Args k{};
  k.n = n;
  k.D = D;
  k.branch = branch;
  k.residual = residual;
  k.gate = gate;
  k.ldu = branch_stride;
  k.ldh = residual_stride;
  k.lda = gate_stride;
  const void* vec[kVectors] = {post_weight, post_bias, scale, next_weight, nullptr};
  for (int i = 0; i < kVectors; ++i) k.vec[i] = vec[i];
  k.g1 = grad_hidden;
  k.g2 = grad_y;
  k.ld1 = grad_hidden_stride;
  k.ld2 = grad_y_stride;
  k.stats = const_cast<float*>(stats);
  k.gu = grad_branch;
  k.gh = grad_residual;
  k.ga = grad_gate;
  k.part = params ? static_cast<float*>(workspace) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using TW = decltype(tw);
    if (n > 0) {
      const int err = with_shape<T>(D, [&](auto WC, auto NC, auto VC) {
        constexpr int W = decltype(WC)::value, NT = decltype(NC)::value, V = decltype(VC)::value;
        return with_form(gate_kind, layer, n * D * static_cast<int64_t>(sizeof(T)) >= kPastBytes, [&](auto GC, auto LC, auto PC) {
          k.nb = bwd_blocks(n, Shape<NT>::kRows, NT);
          hipLaunchKernelGGL((bwd_kernel<T, TW, W, NT, V, decltype(GC)::value, decltype(LC)::value,
                                        decltype(PC)::value>), dim3(k.nb),
                             dim3(Shape<NT>::kThreads), 0, st, k);
          return check_launch(who);
        });
      });
      if (err) return err;
    }
    if (!params) return static_cast<int>(kOk);
    hipLaunchKernelGGL((param_kernel<TW>), dim3((D + kParamCols - 1) / kParamCols, kVectors), dim3(kParamThreads), 0, st,
                       k.part, k.nb, D, outs);
    return check_launch(who);
  });
}

}  // extern "C"

// LayerNorm of rows of 1 <= D <= 16384 values, float32 or bf16, forward and
// backward: the model's output norm (width hidden * (layers + 1)) and any other
// norm beyond the 256 values of the block ops (nodeops.hip).
//
// Row x, xh = (x - mean) rstd, y = xh w + b. Backward, with d = g w:
//   grad_x = rstd (d - mean(d) - xh mean(d xh)),
//   grad_w = sum over rows of g xh, grad_b = sum over rows of g.
//
// Both passes are streams: the forward reads a row once and writes it once, the
// backward reads x and g once and writes grad_x; a row stays in registers
// between its sums and its results (the variance is that of the centred
// values), and the next row's loads are issued before the current row's sums.
// NT threads own a row: lanes of a wavefront while the registers of 64 lanes
// hold it, a workgroup beyond. The parameter gradients are added up per thread
// over the rows of its workgroup, one partial row a workgroup, which
// param_kernel adds in a fixed order (no atomics).
//
// HBM bounds all of it (a copy of 4 GiB moves 4.75 TB/s here, a fill 6.85; the
// VALU is 47 to 67% busy). Measured, forward / backward / parameters:
//   16,384 x 8192 bf16   88 us (6.1 TB/s) / 143 (5.6) / 5
//   24,492 x 1280 f32    37 us (6.8 TB/s) /  58 (6.5) / 4
//   10,007 x 1001 bf16   11 us (3.6 TB/s) /  15 (4.1) / 3.5, one to two waves of
//                        workgroups: latency
//   one row of 4096      2.4 us, a launch and two reductions
#include "rowops.h"
#include "rowvec.h"

namespace cign {
namespace layernorm {
using namespace rowvec;

constexpr int kMaxWidth = 16384;

template <int N>
using IC = std::integral_constant<int, N>;

template <int NT>
struct Shape {
  static constexpr int kThreads = NT < kBlock ? kBlock : NT;
  static constexpr int kRows = kThreads / NT;                          // rows of a workgroup at a time
  static constexpr int kSlots = NT > kWave ? 2 * (NT / kWave) : 1;     // LDS slots of its reductions
};

// A chunk's own values of a result: whole chunks, value by value at a ragged end.
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

// Rows r, r + step, ...: y, and the statistics that the backward takes. The
// parameters stay in registers as they are stored, since every row needs them.
template <typename T, typename TW, int W, int NT, int V, bool PAST>
__global__ __launch_bounds__(Shape<NT>::kThreads) void fwd_kernel(int64_t n, int D, const T* x, int64_t ldx,
                                                                  const TW* weight, const TW* bias, float eps, T* y,
                                                                  float* mean, float* rstd) {
  using X = RowChunk<T, W>;
  using P = RowChunk<TW, W>;
  __shared__ float slots[Shape<NT>::kSlots][1];
  GroupReduce<NT, 1> reduce(slots);
  const int q = threadIdx.x & (NT - 1);
  int at[V], own[V];
  typename P::Raw wr[V], br[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = q + v * NT;
    at[v] = chunk_start<W>(c, D);
    own[v] = c * W - at[v];
    if (weight) wr[v] = P::load(weight + at[v]);
    if (bias) br[v] = P::load(bias + at[v]);
  }
  const float inv = 1.0f / static_cast<float>(D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * Shape<NT>::kRows;
  int64_t r = static_cast<int64_t>(blockIdx.x) * Shape<NT>::kRows + threadIdx.x / NT;
  typename X::Raw next[V];
  if (r < n)
#pragma unroll
    for (int v = 0; v < V; ++v) next[v] = X::load(x + r * ldx + at[v]);
  for (; r < n; r += step) {
    float xv[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v) X::unpack(next[v], xv[v]);
    const int64_t rn = r + step < n ? r + step : r;
#pragma unroll
    for (int v = 0; v < V; ++v) next[v] = X::load(x + rn * ldx + at[v]);
    float s[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int w = 0; w < W; ++w) s[0] += w >= own[v] ? xv[v][w] : 0.0f;
    reduce.sum(s);
    const float mu = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        xv[v][w] -= mu;
        s[0] += w >= own[v] ? xv[v][w] * xv[v][w] : 0.0f;
      }
    reduce.sum(s);
    const float rs = 1.0f / sqrtf(s[0] * inv + eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (own[v] >= W) continue;
      float o[W], p[W];
#pragma unroll
      for (int w = 0; w < W; ++w) o[w] = xv[v][w] * rs;
      if (weight) {
        P::unpack(wr[v], p);
#pragma unroll
        for (int w = 0; w < W; ++w) o[w] *= p[w];
      }
      if (bias) {
        P::unpack(br[v], p);
#pragma unroll
        for (int w = 0; w < W; ++w) o[w] += p[w];
      }
      store_own<T, W, PAST>(y + r * D, at[v], own[v], o);
    }
    if (q == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

// grad_x of a workgroup's rows, and its part of the parameters' gradients:
// part [2][nb][D] (weight, bias).
template <typename T, typename TW, int W, int NT, int V, bool PAST>
__global__ __launch_bounds__(Shape<NT>::kThreads) void bwd_kernel(int64_t n, int D, const T* gy, int64_t ldg,
                                                                  const T* x, int64_t ldx, const TW* weight,
                                                                  const float* mean, const float* rstd, T* gx,
                                                                  float* part, int nb) {
  using X = RowChunk<T, W>;
  using P = RowChunk<TW, W>;
  constexpr int kRows = Shape<NT>::kRows;
  __shared__ float slots[Shape<NT>::kSlots][2];
  GroupReduce<NT, 2> reduce(slots);
  const int q = threadIdx.x & (NT - 1);
  const int slot = threadIdx.x / NT;
  int at[V], own[V];
  typename P::Raw wr[V];
  float aw[V][W], ab[V][W];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = q + v * NT;
    at[v] = chunk_start<W>(c, D);
    own[v] = c * W - at[v];
    if (weight) wr[v] = P::load(weight + at[v]);
#pragma unroll
    for (int w = 0; w < W; ++w) aw[v][w] = ab[v][w] = 0.0f;
  }
  const float inv = 1.0f / static_cast<float>(D);
  // The next row's loads go out before this row's sums, except by 1024 threads,
  // whose 128 registers do not hold both. Workgroups take every nb-th group of
  // rows: blocks of rows lie 1 MB apart where the rows' bytes are a power of two,
  // on the same memory channels at a time (6144 float32 columns, 268 MB: 205 us in
  // blocks, 140 so; 1200: 178 and 146). Rows of 1024 threads, one at a time, do
  // better in blocks (16384 columns: 150 and 166).
  constexpr bool kAhead = NT < 1024;
  const int64_t step = kAhead ? static_cast<int64_t>(nb) * kRows : kRows;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows, r1 = n;
  if (!kAhead) rowops::block_rows(n, nb, blockIdx.x, r0, r1);
  int64_t r = r0 + slot;
  typename X::Raw xn[V], gn[V];
  float mun = 0.0f, rsn = 0.0f;
  const auto load = [&](int64_t row) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      xn[v] = X::load(x + row * ldx + at[v]);
      gn[v] = X::load(gy + row * ldg + at[v]);
    }
    mun = mean[row];
    rsn = rstd[row];
  };
  if (kAhead && r < r1) load(r);
  for (; r < r1; r += step) {
    if (!kAhead) load(r);
    float xh[V][W], g[V][W];
    const float mu = mun, rs = rsn;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      X::unpack(xn[v], xh[v]);
      X::unpack(gn[v], g[v]);
    }
    if (kAhead) load(r + step < r1 ? r + step : r);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p[W];
      if (weight) {
        P::unpack(wr[v], p);
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w) p[w] = 1.0f;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        xh[v][w] = (xh[v][w] - mu) * rs;
        aw[v][w] = fmaf(g[v][w], xh[v][w], aw[v][w]);
        ab[v][w] += g[v][w];
        g[v][w] *= p[w];
        s[0] += w >= own[v] ? g[v][w] : 0.0f;
        s[1] += w >= own[v] ? g[v][w] * xh[v][w] : 0.0f;
      }
    }
    if (!gx) continue;  // only the parameters' gradients are asked for
    reduce.sum(s);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (own[v] >= W) continue;
      float o[W];
#pragma unroll
      for (int w = 0; w < W; ++w) o[w] = rs * (g[v][w] - c1 - xh[v][w] * c2);
      store_own<T, W, PAST>(gx + r * D, at[v], own[v], o);
    }
  }
  if (!part) return;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (own[v] >= W) continue;
      store_own<float, W, false>(part + static_cast<int64_t>(blockIdx.x) * D, at[v], own[v], aw[v]);
      store_own<float, W, false>(part + (static_cast<int64_t>(nb) + blockIdx.x) * D, at[v], own[v], ab[v]);
    }
  } else {
    // the workgroup's row slots, added in order
    constexpr int kCells = NT * V * W;
    __shared__ float lds[kRows * kCells];
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int w = 0; w < W; ++w) lds[slot * kCells + (q + v * NT) * W + w] = k ? ab[v][w] : aw[v][w];
      __syncthreads();
      float* dst = part + (static_cast<int64_t>(k) * nb + blockIdx.x) * D;
      for (int i = threadIdx.x; i < kCells; i += kBlock) {
        const int c = i / W;
        const int col = chunk_start<W>(c, D) + i % W;
        if (c * W >= D || col < c * W) continue;  // past the row, or another chunk's
        float s = 0.0f;
        for (int j = 0; j < kRows; ++j) s += lds[j * kCells + i];
        dst[col] = s;
      }
    }
  }
}

// grad_w and grad_b from the nb partial rows of each: a workgroup adds 32
// columns, 32 slices of the partial rows at a time, then the slices in an LDS
// tree; a fixed order. 2 x 256 x 8192 floats (17 MB) 5 us = 3.4 TB/s, from the
// cache that bwd_kernel left them in; bounded by its launch and eight to sixteen
// dependent steps.
constexpr int kParamCols = 32, kParamThreads = 1024;

template <typename TW>
__global__ __launch_bounds__(kParamThreads) void param_kernel(const float* part, int nb, int D, TW* gw, TW* gb) {
  constexpr int kSlices = kParamThreads / kParamCols;
  __shared__ float red[kParamThreads];
  TW* out = blockIdx.y == 0 ? gw : gb;
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

// f(IC<W>, IC<NT>, IC<V>) for rows of D values of T: the lanes of a row are the
// next power of two of its chunks, 64 lanes hold up to five chunks of float32
// each or four of bf16 (backward of 1,200 bf16 columns, 134 MB: 66 us against 102
// by 256 threads of one chunk, 150 of them at work; of 1,600: 76 and 84), wider
// rows take a workgroup of 256, 512 or 1024 threads. 512 threads go as far as
// their registers hold the next row's values too: up to 12,288 columns (backward of
// 11,000 float32 columns, 268 MB: 146 us against 198 by 1024 threads, of bf16 67
// against 98; with 8 and 4 chunks a thread at 16,384 columns 316 and 101 us
// against 151 and 78 by 1024 threads, which spill too, 56 and 20 bytes of their 128
// registers each, but hold one row at a time).
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
  if (nc <= 1) return f(IC<W>(), IC<1>(), IC<1>());
  if (nc <= 2) return f(IC<W>(), IC<2>(), IC<1>());
  if (nc <= 4) return f(IC<W>(), IC<4>(), IC<1>());
  if (nc <= 8) return f(IC<W>(), IC<8>(), IC<1>());
  if (nc <= 16) return f(IC<W>(), IC<16>(), IC<1>());
  if (nc <= 32) return f(IC<W>(), IC<32>(), IC<1>());
  if (nc <= 64) return f(IC<W>(), IC<64>(), IC<1>());
  if (nc <= 128) return f(IC<W>(), IC<64>(), IC<2>());
  if (nc <= 192) return f(IC<W>(), IC<64>(), IC<3>());
  if (nc <= 256) return f(IC<W>(), IC<64>(), IC<4>());
  if constexpr (W == 4)
    if (nc <= 320) return f(IC<W>(), IC<64>(), IC<5>());
  if (nc <= 512) return f(IC<W>(), IC<256>(), IC<2>());
  if constexpr (W == 4) {
    if (nc <= 768) return f(IC<W>(), IC<256>(), IC<3>());
    if (nc <= 1024) return f(IC<W>(), IC<256>(), IC<4>());
    if (nc <= 2048) return f(IC<W>(), IC<512>(), IC<4>());
    if (nc <= 512 * 6) return f(IC<W>(), IC<512>(), IC<6>());
    return f(IC<W>(), IC<1024>(), IC<4>());
  } else {
    if (nc <= 1024) return f(IC<W>(), IC<512>(), IC<2>());
    if (nc <= 1536) return f(IC<W>(), IC<512>(), IC<3>());
    return f(IC<W>(), IC<1024>(), IC<2>());
  }
}

// f(T, TW) for the storage codes of rows and parameters.
template <class F>
int with_types(int x_dtype, int w_dtype, F&& f) {
  if (x_dtype == kF32) return f(float(), float());
  if (w_dtype == kF32) return f(bf16(), float());
  return f(bf16(), bf16());
}

int check_args(const char* who, int64_t n, int D, int x_dtype, int w_dtype) {
  if (n < 0) return set_error(kInvalid, "%s: negative row count", who);
  if (D < 1 || D > kMaxWidth) return set_error(kInvalid, "%s: requires 1<=D<=%d, got %d", who, kMaxWidth, D);
  if ((x_dtype != kF32 && x_dtype != kBF16) || (w_dtype != kF32 && w_dtype != x_dtype))
    return set_error(kInvalid, "%s: dtypes are 0 or 1, the parameters' 0 or the rows'", who);
  return kOk;
}

// Workgroups of the backward, its partial rows: what the card holds at a time
// for rows of 512 threads and more (16,384 rows of 8192 bf16 142 + 5 us, 146 + 8
// by 512), two a CU for the others (10,007 rows of 1001 bf16 14.5 us, 17 by 256 or
// 1024; 22,369 of 3000 69, 90 and 80).
int bwd_blocks(int64_t n, int rows, int threads) {
  const int64_t groups = (n + rows - 1) / rows, most = threads >= 512 ? 256 : 512;
  return static_cast<int>(groups < most ? groups : most);
}

// Results of this many bytes and more are written past the cache (rowvec.h):
// forward and backward of 125 MB take 99 us instead of 118, of 268 MB 256
// instead of 273. With a kernel that reads each result at once: 96 MB 2%
// slower, 125 MB 198 us instead of 218, 268 MB 454 instead of 438.
constexpr int64_t kPastBytes = 112ll << 20;

}  // namespace layernorm
}  // namespace cign

using namespace cign;
using namespace cign::layernorm;

extern "C" {

int cign_layernorm_fwd(void* stream, int64_t n, int32_t D, int32_t x_dtype, int32_t w_dtype, const void* x,
                       int64_t x_stride, const void* weight, const void* bias, float eps, void* y, float* mean,
                       float* rstd) {
  const char* who = "cign_layernorm_fwd";
  const int rc = check_args(who, n, D, x_dtype, w_dtype);
  if (rc) return rc;
  if (n == 0) return kOk;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return set_error(kInvalid, "%s: null argument", who);
  if (x_stride < 0) return set_error(kInvalid, "%s: negative row stride", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using TW = decltype(tw);
    return with_shape<T>(D, [&](auto WC, auto NC, auto VC) {
      constexpr int W = decltype(WC)::value, NT = decltype(NC)::value, V = decltype(VC)::value;
      const int64_t groups = (n + Shape<NT>::kRows - 1) / Shape<NT>::kRows;
      const int grid = static_cast<int>(groups < 2048 ? groups : 2048);
      const auto launch = [&](auto PC) {
        hipLaunchKernelGGL((fwd_kernel<T, TW, W, NT, V, decltype(PC)::value>), dim3(grid), dim3(Shape<NT>::kThreads), 0,
                           st, n, D, static_cast<const T*>(x), x_stride, static_cast<const TW*>(weight),
                           static_cast<const TW*>(bias), eps, static_cast<T*>(y), mean, rstd);
      };
      n * D * static_cast<int64_t>(sizeof(T)) >= kPastBytes ? launch(std::true_type()) : launch(std::false_type());
      return check_launch(who);
    });
  });
}

int64_t cign_layernorm_bwd_workspace_bytes(int64_t n, int32_t D) {
  if (n < 0 || D < 1 || D > kMaxWidth) return 0;
  return 2 * static_cast<int64_t>(sizeof(float)) * bwd_blocks(n, 1, 1) * D;
}

int cign_layernorm_bwd(void* stream, int64_t n, int32_t D, int32_t x_dtype, int32_t w_dtype, const void* grad_y,
                       int64_t grad_y_stride, const void* x, int64_t x_stride, const void* weight, const float* mean,
                       const float* rstd, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                       int64_t workspace_bytes) {
  const char* who = "cign_layernorm_bwd";
  const int rc = check_args(who, n, D, x_dtype, w_dtype);
  if (rc) return rc;
  if (n > 0 && (!grad_y || !x || !mean || !rstd)) return set_error(kInvalid, "%s: null argument", who);
  if (x_stride < 0 || grad_y_stride < 0) return set_error(kInvalid, "%s: negative row stride", who);
  const bool params = grad_weight || grad_bias;
  if (!params && (!grad_x || n == 0)) return kOk;
  if (params && (!workspace || workspace_bytes < cign_layernorm_bwd_workspace_bytes(n, D)))
    if (n > 0) return set_error(kInvalid, "%s: workspace too small", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_types(x_dtype, w_dtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using TW = decltype(tw);
    float* part = params ? static_cast<float*>(workspace) : nullptr;
    int nb = 0;
    if (n > 0) {
      const int err = with_shape<T>(D, [&](auto WC, auto NC, auto VC) {
        constexpr int W = decltype(WC)::value, NT = decltype(NC)::value, V = decltype(VC)::value;
        nb = bwd_blocks(n, Shape<NT>::kRows, NT);
        const auto launch = [&](auto PC) {
          hipLaunchKernelGGL((bwd_kernel<T, TW, W, NT, V, decltype(PC)::value>), dim3(nb), dim3(Shape<NT>::kThreads), 0,
                             st, n, D, static_cast<const T*>(grad_y), grad_y_stride, static_cast<const T*>(x), x_stride,
                             static_cast<const TW*>(weight), mean, rstd, static_cast<T*>(grad_x), part, nb);
        };
        n * D * static_cast<int64_t>(sizeof(T)) >= kPastBytes ? launch(std::true_type()) : launch(std::false_type());
        return check_launch(who);
      });
      if (err) return err;
    }
    if (!params) return static_cast<int>(kOk);
    // no rows: nb = 0 and the sums are zero
    hipLaunchKernelGGL((param_kernel<TW>), dim3((D + kParamCols - 1) / kParamCols, 2), dim3(kParamThreads), 0, st, part,
                       nb, D, static_cast<TW*>(grad_weight), static_cast<TW*>(grad_bias));
    return check_launch(who);
  });
}

}  // extern "C"

// The global norm of many tensors, sqrt(sum of all squares), and the tensors
// scaled by min(1, max_norm / (norm + 1e-6)): the clipping of a training step.
//
// Tensors are read as flat runs of values, float32 or bf16, in chunks of one tensor
// each; the table of tensors travels in the kernel's arguments, 128 of them a launch,
// so that nothing is copied to the device. A workgroup adds its chunk's squares in
// float64, where no gradient over- or underflows (the VALU multiplies float64 at half
// of float32's rate here, and is about half busy), and stores one partial sum; the
// scaling kernel's workgroups each add the partial sums up in one order and scale
// their chunk. No atomics: the same bits in every run.
//
// HBM bounds the large ones: 500,000,000 bf16 in 200 tensors, the norm 182 us (5.5
// TB/s), clipped into one packed buffer 562 us (3 GB, 5.3 TB/s; a copy moves 4.75).
// Launches bound the small ones: 62 tensors of 2,600,000 float32 in all 8 us and 12.5.
#include <algorithm>

#include "rowvec.h"

namespace cign {
namespace gradnorm {
using rowvec::RowChunk;

constexpr int kTable = 128;       // tensors of a launch
constexpr int kGroups = 1536, kManyGroups = 4096;  // chunks aimed at
constexpr int64_t kLeast = 8192, kMost = 32768;  // values of a chunk: at least; beyond, more chunks

// Tensors of this many bytes and more are scaled from the last to the first and
// written past the cache (1 GB of bf16 562 us, 597 through the cache, 588 in order);
// what is smaller stays in it for the optimizer.
constexpr int64_t kLargeBytes = 192ll << 20;

struct Table {
  const void* p[kTable];
  void* out[kTable];
  int64_t n[kTable];
  int32_t first[kTable + 1];  // first chunk of a tensor, in the launch
  uint8_t bf16[kTable];
  int32_t count;
};

struct Part {
  int t;
  int64_t from, to;
};

// The workgroup's tensor: the last one whose first chunk is not behind it, by a vote
// over the table's two halves (a search would be seven loads behind each other).
__device__ __forceinline__ Part part_of(const Table& table, int64_t chunk, int b) {
  const int l = lane_id();
  const int lo = l < table.count && table.first[l] <= b, hi = l + 64 < table.count && table.first[l + 64] <= b;
  const int t = __popcll(__ballot(lo)) + __popcll(__ballot(hi)) - 1;
  const int64_t from = static_cast<int64_t>(b - table.first[t]) * chunk;
  return Part{t, from, min(from + chunk, table.n[t])};
}

// The sum of v over the workgroup, in every thread.
__device__ __forceinline__ double group_sum(double v, double* lds) {
  for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o, kWave);
  if (lane_id() == 0) lds[wave_id()] = v;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int i = 1; i < kWavesPerBlock; ++i) s += lds[i];
  return s;
}

template <typename T>
__device__ __forceinline__ double squares(const T* p, int64_t from, int64_t to) {
  constexpr int W = rowvec::kChunk<T>, U = 4;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t i = from + threadIdx.x * W;
  for (; i + (U - 1) * W * kBlock + W <= to; i += U * W * kBlock) {
    typename RowChunk<T, W>::Raw q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = RowChunk<T, W>::load(p + i + u * W * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[W];
      RowChunk<T, W>::unpack(q[u], v);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k & 3] = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), acc[k & 3]);
    }
  }
  for (; i < to; i += W * kBlock)
    for (int k = 0; k < W && i + k < to; ++k) {
      const double v = to_f32(p[i + k]);
      acc[0] = fma(v, v, acc[0]);
    }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__global__ __launch_bounds__(kBlock) void squares_kernel(Table table, int64_t chunk, double* part) {
  __shared__ double lds[kWavesPerBlock];
  const Part c = part_of(table, chunk, blockIdx.x);
  const double mine = table.bf16[c.t] ? squares(static_cast<const bf16*>(table.p[c.t]), c.from, c.to)
                                      : squares(static_cast<const float*>(table.p[c.t]), c.from, c.to);
  const double s = group_sum(mine, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double* part, int parts, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kBlock) s += part[i];
  return sqrt(group_sum(s, lds));
}

__global__ __launch_bounds__(kBlock) void norm_kernel(const double* part, int parts, float* norm) {
  __shared__ double lds[kWavesPerBlock];
  const double v = norm_of(part, parts, lds);
  if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

// out = p by `by`, of the chunk's values; all chunks are moved on to where out's lines
// of 128 bytes begin (a packed buffer's tensors lie anywhere), so that stores are
// whole lines and only loads are not aligned.
template <bool PAST, typename T>
__device__ __forceinline__ void scale(const T* p, T* out, int64_t from, int64_t to, int64_t n, float by) {
  constexpr int W = rowvec::kChunk<T>, U = 4;
  const int head = static_cast<int>(-(reinterpret_cast<uintptr_t>(out) / sizeof(T)) & (128 / sizeof(T) - 1));
  const int64_t begin = from == 0 ? min(static_cast<int64_t>(head), n) : min(from + head, n);
  if (from == 0 && threadIdx.x < begin) out[threadIdx.x] = from_f32<T>(to_f32(p[threadIdx.x]) * by);
  to = to == n ? n : min(to + head, n);
  int64_t i = begin + threadIdx.x * W;
  for (; i + (U - 1) * W * kBlock + W <= to; i += U * W * kBlock) {
    typename RowChunk<T, W>::Raw q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = RowChunk<T, W>::load(p + i + u * W * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[W];
      RowChunk<T, W>::unpack(q[u], v);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] *= by;
      if constexpr (PAST) RowChunk<T, W>::store_past(out + i + u * W * kBlock, v);
      else RowChunk<T, W>::store(out + i + u * W * kBlock, v);
    }
  }
  for (; i < to; i += W * kBlock)
    for (int k = 0; k < W && i + k < to; ++k) out[i + k] = from_f32<T>(to_f32(p[i + k]) * by);
}

// LARGE: from the last chunk to the first, the squares' pass having left the last ones
// in the 256 MB cache, and stores past it.
template <bool LARGE>
__global__ __launch_bounds__(kBlock) void scale_kernel(Table table, int64_t chunk, const double* part, int parts,
                                                       float max_norm, float* norm) {
  __shared__ double lds[kWavesPerBlock];
  const double total = norm_of(part, parts, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
  double by = static_cast<double>(max_norm) / (total + 1e-6);
  if (by > 1.0) by = 1.0;  // a NaN stays
  const Part c = part_of(table, chunk, LARGE ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  if (by == 1.0 && table.out[c.t] == table.p[c.t]) return;
  if (table.bf16[c.t])
    scale<LARGE>(static_cast<const bf16*>(table.p[c.t]), static_cast<bf16*>(table.out[c.t]), c.from, c.to, table.n[c.t],
                 static_cast<float>(by));
  else
    scale<LARGE>(static_cast<const float*>(table.p[c.t]), static_cast<float*>(table.out[c.t]), c.from, c.to, table.n[c.t],
                 static_cast<float>(by));
}

// Values of a chunk, and the chunks of all tensors; a multiple of 8 so that every
// chunk of a tensor has its first one's alignment.
int64_t chunk_of(int32_t count, const int64_t* sizes, int64_t* chunks) {
  int64_t total = 0;
  for (int32_t i = 0; i < count; ++i) total += sizes[i];
  const auto share = [&](int64_t groups) { return (total + groups - 1) / groups; };
  const int64_t want = std::max(kLeast, std::min(share(kGroups), std::max(kMost, share(kManyGroups))));
  const int64_t chunk = (want + 2047) / 2048 * 2048;
  *chunks = 0;
  for (int32_t i = 0; i < count; ++i) *chunks += (sizes[i] + chunk - 1) / chunk;
  return chunk;
}

int check_tensors(const char* who, int32_t count, const void* const* grads, const int64_t* sizes,
                  const int32_t* dtypes) {
  if (count < 0) return set_error(kInvalid, "%s: negative count", who);
  if (count > 0 && (!grads || !sizes || !dtypes)) return set_error(kInvalid, "%s: null argument", who);
  for (int32_t i = 0; i < count; ++i) {
    if (sizes[i] < 0) return set_error(kInvalid, "%s: negative size of tensor %d", who, i);
    if (sizes[i] > 0 && !grads[i]) return set_error(kInvalid, "%s: tensor %d is null", who, i);
    if (dtypes[i] != kF32 && dtypes[i] != kBF16) return set_error(kInvalid, "%s: dtypes are 0 or 1", who);
  }
  return kOk;
}

// f(table, blocks, chunks before) for runs of up to kTable tensors that are not empty,
// or from the last run to the first.
template <class F>
int for_tables(int32_t count, const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes,
               int64_t chunk, bool backwards, F&& f) {
  int32_t full = 0;
  for (int32_t i = 0; i < count; ++i) full += sizes[i] > 0;
  const int32_t runs = (full + kTable - 1) / kTable;
  for (int32_t r = 0; r < runs; ++r) {
    const int32_t run = backwards ? runs - 1 - r : r;
    Table t;
    t.count = 0;
    t.first[0] = 0;
    int32_t before = 0, seen = 0;
    for (int32_t i = 0; i < count; ++i) {
      if (sizes[i] == 0) continue;
      const int32_t chunks = static_cast<int32_t>((sizes[i] + chunk - 1) / chunk), at = seen++ / kTable;
      if (at < run) before += chunks;
      if (at != run) continue;
      const int k = t.count++;
      t.p[k] = grads[i];
      t.out[k] = out ? out[i] : nullptr;
      t.n[k] = sizes[i];
      t.bf16[k] = dtypes[i] == kBF16;
      t.first[k + 1] = t.first[k] + chunks;
    }
    if (const int rc = f(t, t.first[t.count], before)) return rc;
  }
  return kOk;
}

int run(const char* who, void* stream, int32_t count, const void* const* grads, const int64_t* sizes,
        const int32_t* dtypes, float max_norm, void* const* out, float* norm, void* workspace,
        int64_t workspace_bytes) {
  int64_t chunks;
  const int64_t chunk = chunk_of(count, sizes, &chunks);
  if (chunks > INT32_MAX) return set_error(kInvalid, "%s: too many tensors", who);
  if (chunks > 0 && (!workspace || workspace_bytes < static_cast<int64_t>(sizeof(double)) * chunks))
    return set_error(kInvalid, "%s: workspace too small", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int parts = static_cast<int>(chunks);
  int rc = for_tables(count, grads, out, sizes, dtypes, chunk, false,
                      [&](const Table& t, int32_t blocks, int32_t before) {
    hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kBlock), 0, st, t, chunk, part + before);
    return check_launch(who);
  });
  if (rc) return rc;
  if (!out || parts == 0) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kBlock), 0, st, part, parts, norm);
    return check_launch(who);
  }
  int64_t bytes = 0;
  for (int32_t i = 0; i < count; ++i) bytes += sizes[i] * (dtypes[i] == kF32 ? 4 : 2);
  const bool large = bytes >= kLargeBytes;
  return for_tables(count, grads, out, sizes, dtypes, chunk, large, [&](const Table& t, int32_t blocks, int32_t) {
    if (large)
      hipLaunchKernelGGL((scale_kernel<true>), dim3(blocks), dim3(kBlock), 0, st, t, chunk, part, parts, max_norm, norm);
    else
      hipLaunchKernelGGL((scale_kernel<false>), dim3(blocks), dim3(kBlock), 0, st, t, chunk, part, parts, max_norm, norm);
    return check_launch(who);
  });
}

}  // namespace gradnorm
}  // namespace cign

using namespace cign;
using namespace cign::gradnorm;

extern "C" {

int64_t cign_grad_norm_workspace_bytes(int32_t count, const int64_t* sizes) {
  if (count <= 0 || !sizes) return 0;
  for (int32_t i = 0; i < count; ++i)
    if (sizes[i] < 0) return 0;
  int64_t chunks;
  chunk_of(count, sizes, &chunks);
  return static_cast<int64_t>(sizeof(double)) * chunks;
}

int cign_grad_norm(void* stream, int32_t count, const void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                   float* norm, void* workspace, int64_t workspace_bytes) {
  const char* who = "cign_grad_norm";
  if (const int rc = check_tensors(who, count, grads, sizes, dtypes)) return rc;
  if (!norm) return set_error(kInvalid, "%s: null argument", who);
  return run(who, stream, count, grads, sizes, dtypes, 0.0f, nullptr, norm, workspace, workspace_bytes);
}

int cign_clip_grad_norm(void* stream, int32_t count, const void* const* grads, const int64_t* sizes,
                        const int32_t* dtypes, float max_norm, void* const* out, float* norm, void* workspace,
                        int64_t workspace_bytes) {
  const char* who = "cign_clip_grad_norm";
  if (const int rc = check_tensors(who, count, grads, sizes, dtypes)) return rc;
  if (!norm || (count > 0 && !out)) return set_error(kInvalid, "%s: null argument", who);
  for (int32_t i = 0; i < count; ++i)
    if (sizes[i] > 0 && !out[i]) return set_error(kInvalid, "%s: output %d is null", who, i);
  if (!(max_norm >= 0.0f)) return set_error(kInvalid, "%s: max_norm must not be negative", who);
  return run(who, stream, count, grads, sizes, dtypes, max_norm, out, norm, workspace, workspace_bytes);
}

}  // extern "C"

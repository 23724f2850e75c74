// The global norm of many tensors, sqrt(sum of all squares), and the tensors
// scaled by min(1, max_norm / (norm + 1e-6)): the clipping of a training step.
//
// Tensors are read as flat runs of values, float32 or bf16, in chunks of one
// tensor each; the table of tensors travels in the kernel's arguments, 128 of them
// a launch, so that nothing is copied to the device. A workgroup adds its chunk's
// squares in float64, where no gradient over- or underflows (the VALU's float64
// rate is half of float32's here), and stores one partial sum; the scaling kernel's workgroups each
// add the partial sums up in one order and scale their chunk. No atomics: the same
// bits in every run.
#include <algorithm>

#include "rowvec.h"

namespace cign {
namespace gradnorm {
using rowvec::RowChunk;

constexpr int kTable = 128;       // tensors of a launch
constexpr int kGroups = 1536;     // chunks aimed at: six workgroups a CU
constexpr int64_t kLeast = 8192;  // values of a chunk at least

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

__device__ __forceinline__ Part part_of(const Table& table, int64_t chunk) {
  int lo = 0, hi = table.count;
  const int b = blockIdx.x;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.first[mid] <= b) lo = mid;
    else hi = mid;
  }
  const int64_t from = static_cast<int64_t>(b - table.first[lo]) * chunk;
  return Part{lo, from, min(from + chunk, table.n[lo])};
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
  constexpr int U = 4;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t i = from + threadIdx.x * 8;
  for (; i + (U - 1) * 8 * kBlock + 8 <= to; i += U * 8 * kBlock) {
    typename RowChunk<T, 8>::Raw q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = RowChunk<T, 8>::load(p + i + u * 8 * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[8];
      RowChunk<T, 8>::unpack(q[u], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k & 3] = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), acc[k & 3]);
    }
  }
  for (; i < to; i += 8 * kBlock)
    for (int k = 0; k < 8 && i + k < to; ++k) {
      const double v = to_f32(p[i + k]);
      acc[0] = fma(v, v, acc[0]);
    }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__global__ __launch_bounds__(kBlock) void squares_kernel(Table table, int64_t chunk, double* part) {
  __shared__ double lds[kWavesPerBlock];
  const Part c = part_of(table, chunk);
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

template <typename T>
__device__ __forceinline__ void scale(const T* p, T* out, int64_t from, int64_t to, float by) {
  constexpr int U = 4;
  int64_t i = from + threadIdx.x * 8;
  for (; i + (U - 1) * 8 * kBlock + 8 <= to; i += U * 8 * kBlock) {
    typename RowChunk<T, 8>::Raw q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = RowChunk<T, 8>::load(p + i + u * 8 * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[8];
      RowChunk<T, 8>::unpack(q[u], v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= by;
      RowChunk<T, 8>::store(out + i + u * 8 * kBlock, v);
    }
  }
  for (; i < to; i += 8 * kBlock)
    for (int k = 0; k < 8 && i + k < to; ++k) out[i + k] = from_f32<T>(to_f32(p[i + k]) * by);
}

__global__ __launch_bounds__(kBlock) void scale_kernel(Table table, int64_t chunk, const double* part, int parts,
                                                       double max_norm, float* norm) {
  __shared__ double lds[kWavesPerBlock];
  const double total = norm_of(part, parts, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
  double by = max_norm / (total + 1e-6);
  if (by > 1.0) by = 1.0;  // a NaN stays
  const Part c = part_of(table, chunk);
  if (by == 1.0 && table.out[c.t] == table.p[c.t]) return;
  if (table.bf16[c.t])
    scale(static_cast<const bf16*>(table.p[c.t]), static_cast<bf16*>(table.out[c.t]), c.from, c.to,
          static_cast<float>(by));
  else
    scale(static_cast<const float*>(table.p[c.t]), static_cast<float*>(table.out[c.t]), c.from, c.to,
          static_cast<float>(by));
}

// Values of a chunk, and the chunks of all tensors; a multiple of 8 so that every
// chunk of a tensor has its first one's alignment.
int64_t chunk_of(int32_t count, const int64_t* sizes, int64_t* chunks) {
  int64_t total = 0;
  for (int32_t i = 0; i < count; ++i) total += sizes[i];
  const int64_t chunk = std::max(kLeast, ((total + kGroups - 1) / kGroups + 2047) / 2048 * 2048);
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

// f(table, blocks, chunks before) for runs of up to kTable tensors that are not empty
template <class F>
int for_tables(int32_t count, const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes,
               int64_t chunk, F&& f) {
  Table t;
  t.count = 0;
  t.first[0] = 0;
  int32_t before = 0;
  for (int32_t i = 0; i <= count; ++i) {
    if (t.count == kTable || (i == count && t.count > 0)) {
      if (const int rc = f(t, t.first[t.count], before)) return rc;
      before += t.first[t.count];
      t.count = 0;
    }
    if (i == count) break;
    if (sizes[i] == 0) continue;
    const int k = t.count++;
    t.p[k] = grads[i];
    t.out[k] = out ? out[i] : nullptr;
    t.n[k] = sizes[i];
    t.bf16[k] = dtypes[i] == kBF16;
    t.first[k + 1] = t.first[k] + static_cast<int32_t>((sizes[i] + chunk - 1) / chunk);
  }
  return kOk;
}

int run(const char* who, void* stream, int32_t count, const void* const* grads, const int64_t* sizes,
        const int32_t* dtypes, double max_norm, void* const* out, float* norm, void* workspace,
        int64_t workspace_bytes) {
  int64_t chunks;
  const int64_t chunk = chunk_of(count, sizes, &chunks);
  if (chunks > INT32_MAX) return set_error(kInvalid, "%s: too many tensors", who);
  if (chunks > 0 && (!workspace || workspace_bytes < static_cast<int64_t>(sizeof(double)) * chunks))
    return set_error(kInvalid, "%s: workspace too small", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int parts = static_cast<int>(chunks);
  int rc = for_tables(count, grads, out, sizes, dtypes, chunk, [&](const Table& t, int32_t blocks, int32_t before) {
    hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kBlock), 0, st, t, chunk, part + before);
    return check_launch(who);
  });
  if (rc) return rc;
  if (!out || parts == 0) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kBlock), 0, st, part, parts, norm);
    return check_launch(who);
  }
  return for_tables(count, grads, out, sizes, dtypes, chunk, [&](const Table& t, int32_t blocks, int32_t) {
    hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(kBlock), 0, st, t, chunk, part, parts, max_norm, norm);
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
  return run(who, stream, count, grads, sizes, dtypes, 0.0, nullptr, norm, workspace, workspace_bytes);
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

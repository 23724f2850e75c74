// The loss of a student's logits against a teacher's top classes, and its
// gradient.
//
// A row's list names up to K classes i with the teacher's log probabilities at
// temperature T (places with a negative index are empty). With q = softmax(x / T)
// over all V classes:
//   renormalised list:  p = softmax over the list,
//     loss = T^2 sum_i p_i (log p_i - log q_i);
//   with the tail:  p_i = e^(listed value), r = max(0, 1 - sum p) and q_rest =
//     the mass q leaves outside the list,
//     loss = T^2 [sum_i p_i (log p_i - log q_i) + r (log r - log q_rest)].
// With A = sum p + r, the gradient of x_j is g T (A q_j - p_j) for a listed
// class and g T (A q_rest - r) q_j / q_rest for the others (r = 0, q_rest = 1
// for a renormalised list): one exponential a class, relative to the statistics
// of the classes outside the list, where A q_rest - r does not cancel in
// float32 and nothing overflows however small q_rest is.
//
// The forward reads the logits once (rowsoftmax.h); with the tail, listed
// classes are marked in a bitmap in LDS and left out of the sums, which a
// subtraction from the whole sum could not recover where the list holds nearly
// all of the mass. What remains is K values a row, which its lanes finish in
// float64: log p - log q is a difference of near values. The backward reads the
// logits, writes the gradient of a class outside the list for every class, and
// after a barrier the listed ones over it.
#include "rowsoftmax.h"

namespace cign {
namespace distill {
using namespace rowsoftmax;

template <typename T>
struct In {
  int64_t n;
  int V;
  const T* x;
  int64_t ld;
  float c;  // log2(e) / T
  double temperature;
  int K;
  const float* t;        // [n, K]
  const int64_t* index;  // [n, K]
};

// What the backward takes of a row.
struct Stats {
  float mb, l2b, cb;  // gradient of a class outside the list: cb 2^((x - mb) c - l2b)
  float m, l2s, a;    // of a listed class: a 2^((x - m) c - l2s) - p
  float pad[2];
};

struct Out {
  float* loss;
  Stats* stats;  // NULL: neither is kept
  float* p;      // [n, K]: the teacher's mass at the place's class, over all places that name it
};

template <int LPR>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

template <int LPR>
__device__ __forceinline__ float lanes_max(float v) {
  for_offsets<1, LPR>([&](auto OC) { v = fmaxf(v, xor_shfl<decltype(OC)::value>(v)); });
  return v;
}

// Row r by LPR lanes (lane q), from the joined statistics (m, s) of the
// classes outside the list (TAIL) or of all classes.
template <typename T, int LPR, bool TAIL>
__device__ void finish(const In<T>& in, const Out& o, int64_t r, int q, float m, float s) {
  const int64_t* index = in.index + r * in.K;
  const float* t = in.t + r * in.K;
  const T* row = in.x + r * in.ld;
  const double inv_t = 1.0 / in.temperature;
  float top = -kInf, top_x = -kInf, any = 0.0f, bad = 0.0f;
  for (int i = q; i < in.K; i += LPR) {
    const int64_t j = index[i];
    if (j < 0) continue;
    any = 1.0f;
    if (j >= in.V) {
      bad = 1.0f;
      continue;
    }
    top = fmaxf(top, t[i]);
    top_x = fmaxf(top_x, to_f32(row[j]));
  }
  top = lanes_max<LPR>(top);
  top_x = lanes_max<LPR>(top_x);
  any = lanes_max<LPR>(any);
  bad = lanes_max<LPR>(bad);

  // the student over all classes: (mt, st)
  double st = s;
  float mt = m;
  double members = 0.0;
  if constexpr (TAIL) {
    mt = shift_of(fmaxf(s == 0.0f ? -kInf : m, top_x));
    double listed = 0.0;
    for (int i = q; i < in.K; i += LPR) {
      const int64_t j = index[i];
      if (j < 0 || j >= in.V) continue;
      bool first = true;
      for (int k = 0; k < i; ++k) first = first && index[k] != j;
      if (!first) continue;
      members += 1.0;
      listed += exp2f((to_f32(row[j]) - mt) * in.c);
    }
    members = lanes_sum<LPR>(members);
    st = (s == 0.0f ? 0.0 : static_cast<double>(s) * exp2(static_cast<double>((m - mt) * in.c))) +
         lanes_sum<LPR>(listed);
  }
  const bool none = st == 0.0;
  const double lz = none ? 0.0 : log(st);

  // the teacher
  double shift = 0.0;  // log p = t - shift
  if constexpr (!TAIL) {
    double total = 0.0;
    for (int i = q; i < in.K; i += LPR)
      if (index[i] >= 0 && index[i] < in.V) total += exp(static_cast<double>(t[i]) - shift_of(top));
    total = lanes_sum<LPR>(total);
    shift = total == 0.0 ? 0.0 : shift_of(top) + log(total);
  }
  double loss = 0.0, mass = 0.0;
  for (int i = q; i < in.K; i += LPR) {
    const int64_t j = index[i];
    double at_class = 0.0;
    if (j >= 0 && j < in.V) {
      const double lp = static_cast<double>(t[i]) - shift;
      const double p = exp(lp);
      if (p != 0.0) {
        const float x = to_f32(row[j]);
        const double lq = none ? -static_cast<double>(kInf) : (static_cast<double>(x) - mt) * inv_t - lz;
        loss += p * (lp - lq);
        mass += p;
      }
      if (o.p) {
        at_class = p;
        for (int k = 0; k < in.K; ++k)
          if (k != i && index[k] == j) at_class += exp(static_cast<double>(t[k]) - shift);
      }
    }
    if (o.p) o.p[r * in.K + i] = static_cast<float>(at_class);
  }
  loss = lanes_sum<LPR>(loss);
  mass = lanes_sum<LPR>(mass);

  double a = mass, cb = mass, lrest = 0.0;
  if constexpr (TAIL) {
    const double left = any != 0.0f && members < in.V ? fmax(0.0, 1.0 - mass) : 0.0;
    lrest = s == 0.0f ? -static_cast<double>(kInf)
                      : (static_cast<double>(m) - mt) * inv_t + log(static_cast<double>(s)) - lz;
    if (left > 0.0) loss += left * (log(left) - lrest);
    a = mass + left;
    cb = a * exp(lrest) - left;
  }
  if (bad != 0.0f) loss = a = cb = __builtin_nan("");
  if (q != 0) return;
  o.loss[r] = static_cast<float>(loss * in.temperature * in.temperature);
  if (o.stats)
    o.stats[r] = Stats{m, s == 0.0f ? kInf : log2f(s), static_cast<float>(cb), mt,
                       none ? kInf : static_cast<float>(lz * 1.4426950408889634), static_cast<float>(a),
                       {0.0f, 0.0f}};
}

// The bits of a share's chunk c (W places from column c W of the bitmap's
// first column) moved to where its values are.
template <int W>
__device__ __forceinline__ uint32_t kill_bits(const uint32_t* bits, int place, int own) {
  const uint32_t listed = bits[place * W >> 5] >> (place * W & 31);
  return ((1u << own) - 1u) | ((listed << own) & ((1u << W) - 1u));
}

// Rows that LPR lanes hold.
template <typename T, int W, int LPR, int U, bool TAIL>
__global__ __launch_bounds__(kBlock) void lanes_kernel(In<T> in, Out o) {
  constexpr int kRows = kBlock / LPR;
  constexpr int kWords = (LPR * U * W + 31) / 32;
  __shared__ uint32_t bitmap[TAIL ? kRows * kWords : 1];
  const int q = threadIdx.x & (LPR - 1);
  const int slot = threadIdx.x / LPR;
  uint32_t* bits = bitmap + (TAIL ? slot * kWords : 0);
  const int nc = (in.V + W - 1) / W;
  Share<T, W, U> sh;
  sh.place(q, LPR, nc, in.V);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < in.n; base += step) {
    const int64_t r = base + slot;
    const bool active = r < in.n;
    if (active) sh.load(in.x + r * in.ld);
    if constexpr (TAIL) {
      __syncthreads();  // the former rows' bits have been read
      for (int i = q; i < kWords; i += LPR) bits[i] = 0;
      __syncthreads();
      if (active)
        for (int i = q; i < in.K; i += LPR) {
          const int64_t j = in.index[r * in.K + i];
          if (j >= 0 && j < in.V) atomicOr(&bits[j >> 5], 1u << (j & 31));
        }
      __syncthreads();
    }
    if (!active) continue;
#pragma unroll
    for (int u = 0; u < U; ++u)
      mask_out<T, W>(sh.raw[u], TAIL ? kill_bits<W>(bits, q + u * LPR, sh.own[u]) : (1u << sh.own[u]) - 1u);
    float m = sh.largest(), s = 0.0f, t = 0.0f;
    sh.template sums<false>(shift_of(m), in.c, s, t);
    join<LPR>(m, s, t, in.c);
    finish<T, LPR, TAIL>(in, o, r, q, m, s);
  }
}

// Slices of long rows: (m, s) to part[r * S + slice], or, with S = 1, the row.
template <typename T, int U, bool TAIL>
__global__ __launch_bounds__(kBlock) void slice_kernel(In<T> in, Out o, Slicing sl, float2* part) {
  constexpr int W = kChunk<T>;
  constexpr int kWords = kBlock * U * W / 32;
  __shared__ float slots[2 * kWavesPerBlock][3];
  __shared__ uint32_t bits[TAIL ? kWords : 1];
  BlockJoin across(slots);
  const int nc = (in.V + W - 1) / W;
  const int64_t items = in.n * sl.S;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / sl.S;
    const int slice = static_cast<int>(item - r * sl.S);
    const int begin = slice * sl.cps, end = min(begin + sl.cps, nc);
    Share<T, W, U> sh;
    sh.place(begin + threadIdx.x, kBlock, end, in.V);
    sh.load(in.x + r * in.ld);
    if constexpr (TAIL) {
      // (the barrier of the former item's join came after its last read)
      for (int i = threadIdx.x; i < kWords; i += kBlock) bits[i] = 0;
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < in.K) {
        const int64_t j = in.index[r * in.K + threadIdx.x] - static_cast<int64_t>(begin) * W;
        if (j >= 0 && j < static_cast<int64_t>(end - begin) * W) atomicOr(&bits[j >> 5], 1u << (j & 31));
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      mask_out<T, W>(sh.raw[u], TAIL ? kill_bits<W>(bits, threadIdx.x + u * kBlock, sh.own[u]) : (1u << sh.own[u]) - 1u);
    float m = sh.largest(), s = 0.0f, t = 0.0f;
    sh.template sums<false>(shift_of(m), in.c, s, t);
    join<kWave>(m, s, t, in.c);
    across.run(m, s, t, in.c);
    if (sl.S == 1) {
      if (threadIdx.x < kWave) finish<T, kWave, TAIL>(in, o, r, threadIdx.x, m, s);
    } else if (threadIdx.x == 0) {
      part[item] = make_float2(s == 0.0f ? -kInf : m, s);
    }
  }
}

// Rows from their slices, a wavefront a row; lane i holds slice i.
template <typename T, bool TAIL>
__global__ __launch_bounds__(kBlock) void join_kernel(In<T> in, Out o, int S, const float2* part) {
  const int lane = lane_id();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWavesPerBlock;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_id(); r < in.n; r += step) {
    const float2 p = lane < S ? part[r * S + lane] : make_float2(-kInf, 0.0f);
    float m = p.x, s = p.y, t = 0.0f;
    join<kWave>(m, s, t, in.c);
    finish<T, kWave, TAIL>(in, o, r, lane, m, s);
  }
}

// grad_x of rows held by LPR threads (lanes, or LPR = 256: the slices of a
// long row). A row without a listed class, or whose g is zero, is zeros,
// whatever its logits hold.
template <typename T, int W, int LPR, int U>
__global__ __launch_bounds__(kBlock) void grad_kernel(In<T> in, int S, int cps, const Stats* stats, const float* p,
                                                      const float* g_loss, float temperature, T* gx) {
  using X = RowChunk<T, W>;
  constexpr int kRows = kBlock / LPR;
  const int q = threadIdx.x & (LPR - 1);
  const int nc = (in.V + W - 1) / W;
  const int64_t items = in.n * S;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < items; base += step) {
    const int64_t item = base + threadIdx.x / LPR;
    const bool active = item < items;
    const int64_t r = !active ? 0 : S == 1 ? item : item / S;
    const int slice = active && S > 1 ? static_cast<int>(item - r * S) : 0;
    const int begin = slice * cps, end = min(begin + cps, nc);
    const Stats st = stats[r];
    const float gt = g_loss[r] * temperature;
    const bool zero = gt == 0.0f || st.a == 0.0f;
    T* row = gx + r * in.V;
    if (active) {
      Share<T, W, U> sh;
      sh.place(begin + q, LPR, end, in.V);
      if (!zero) sh.load(in.x + r * in.ld);
      const float cb = gt * st.cb;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[W];
        if (zero) {
#pragma unroll
          for (int w = 0; w < W; ++w) v[w] = 0.0f;
        } else {
          X::unpack(sh.raw[u], v);
#pragma unroll
          for (int w = 0; w < W; ++w) v[w] = cb * __builtin_amdgcn_exp2f(fmaf(v[w] - st.mb, in.c, -st.l2b));
        }
        Share<T, W, U>::store(row, sh.at[u], sh.own[u], v);
      }
    }
    __syncthreads();  // the listed classes are written over what another thread of this workgroup stored
    if (active && !zero)
      for (int i = q; i < in.K; i += LPR) {
        const int64_t j = in.index[r * in.K + i];
        if (j < static_cast<int64_t>(begin) * W || j >= static_cast<int64_t>(end) * W || j >= in.V) continue;
        const float x = to_f32(in.x[r * in.ld + j]);
        row[j] = from_f32<T>(gt * (st.a * __builtin_amdgcn_exp2f(fmaf(x - st.m, in.c, -st.l2s)) - p[r * in.K + i]));
      }
  }
}

int check_args(const char* who, int dtype, int64_t n, int V, int64_t ld, int K, float temperature) {
  if (dtype != kF32 && dtype != kBF16) return set_error(kInvalid, "%s: dtype must be 0 or 1", who);
  if (n < 0) return set_error(kInvalid, "%s: negative row count", who);
  if (V < 1 || V > kMaxClasses) return set_error(kInvalid, "%s: requires 1<=V<=%d, got %d", who, kMaxClasses, V);
  if (K < 1 || K > kMaxList) return set_error(kInvalid, "%s: requires 1<=K<=%d, got %d", who, kMaxList, K);
  if (ld < 0) return set_error(kInvalid, "%s: negative row stride", who);
  if (!(temperature > 0.0f && temperature < kInf)) return set_error(kInvalid, "%s: temperature must be positive", who);
  return kOk;
}

template <typename F>
int with_type(int dtype, F&& f) {
  return dtype == kF32 ? f(float()) : f(bf16());
}

template <typename T>
In<T> input(int64_t n, int V, const void* x, int64_t ld, float temperature, int K, const float* t,
            const int64_t* index) {
  return In<T>{n, V, static_cast<const T*>(x), ld, kLog2e / temperature, temperature, K, t, index};
}

template <typename T>
int64_t workspace_bytes(int64_t n, int V) {
  if (wavefront_row<T>(V)) return 0;
  const Slicing sl = slicing<T>(V, n);
  return sl.S == 1 ? 0 : n * sl.S * static_cast<int64_t>(sizeof(float2));
}

template <typename T, bool TAIL>
int forward(const char* who, hipStream_t st, const In<T>& in, const Out& o, void* workspace, int64_t bytes) {
  if (bytes < workspace_bytes<T>(in.n, in.V)) return set_error(kInvalid, "%s: workspace too small", who);
  if (wavefront_row<T>(in.V))
    return with_lanes<T>(in.V, [&](auto WC, auto LC, auto UC) {
      constexpr int W = decltype(WC)::value, LPR = decltype(LC)::value, U = decltype(UC)::value;
      constexpr int kRows = kBlock / LPR;
      hipLaunchKernelGGL((lanes_kernel<T, W, LPR, U, TAIL>), dim3(grid_of((in.n + kRows - 1) / kRows)), dim3(kBlock), 0,
                         st, in, o);
      return check_launch(who);
    });
  const Slicing sl = slicing<T>(in.V, in.n);
  float2* part = static_cast<float2*>(workspace);
  const int rc = with_chunks<T>(sl.U, [&](auto UC) {
    constexpr int U = decltype(UC)::value;
    hipLaunchKernelGGL((slice_kernel<T, U, TAIL>), dim3(grid_of(in.n * sl.S)), dim3(kBlock), 0, st, in, o, sl, part);
    return check_launch(who);
  });
  if (rc || sl.S == 1) return rc;
  hipLaunchKernelGGL((join_kernel<T, TAIL>), dim3(grid_of((in.n + kWavesPerBlock - 1) / kWavesPerBlock)), dim3(kBlock),
                     0, st, in, o, sl.S, part);
  return check_launch(who);
}

}  // namespace distill
}  // namespace cign

using namespace cign;
using namespace cign::distill;

extern "C" {

int64_t cign_distill_topk_workspace_bytes(int32_t dtype, int64_t n, int32_t V) {
  if (n < 1 || V < 1 || V > kMaxClasses) return 0;
  return with_type(dtype, [&](auto t) { return workspace_bytes<decltype(t)>(n, V); });
}

int cign_distill_topk_fwd(void* stream, int32_t dtype, int64_t n, int32_t V, const void* x, int64_t x_stride,
                          float temperature, int32_t tail, int32_t K, const float* teacher_logprob,
                          const int64_t* teacher_index, float* loss, float* stats, float* teacher_mass,
                          void* workspace, int64_t workspace_bytes) {
  const char* who = "cign_distill_topk_fwd";
  const int rc = check_args(who, dtype, n, V, x_stride, K, temperature);
  if (rc) return rc;
  if (n == 0) return kOk;
  if (!x || !teacher_logprob || !teacher_index || !loss || (stats == nullptr) != (teacher_mass == nullptr))
    return set_error(kInvalid, "%s: null argument", who);
  const Out o{loss, reinterpret_cast<Stats*>(stats), teacher_mass};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const In<T> in = input<T>(n, V, x, x_stride, temperature, K, teacher_logprob, teacher_index);
    return tail ? forward<T, true>(who, st, in, o, workspace, workspace_bytes)
                : forward<T, false>(who, st, in, o, workspace, workspace_bytes);
  });
}

int cign_distill_topk_bwd(void* stream, int32_t dtype, int64_t n, int32_t V, const void* x, int64_t x_stride,
                          float temperature, int32_t K, const int64_t* teacher_index, const float* stats,
                          const float* teacher_mass, const float* grad_loss, void* grad_x) {
  const char* who = "cign_distill_topk_bwd";
  const int rc = check_args(who, dtype, n, V, x_stride, K, temperature);
  if (rc) return rc;
  if (n == 0) return kOk;
  if (!x || !teacher_index || !stats || !teacher_mass || !grad_loss || !grad_x)
    return set_error(kInvalid, "%s: null argument", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const In<T> in = input<T>(n, V, x, x_stride, temperature, K, nullptr, teacher_index);
    const auto launch = [&](auto WC, auto LC, auto UC, int S, int cps) {
      constexpr int W = decltype(WC)::value, LPR = decltype(LC)::value, U = decltype(UC)::value;
      constexpr int kRows = kBlock / LPR;
      hipLaunchKernelGGL((grad_kernel<T, W, LPR, U>), dim3(grid_of((n * S + kRows - 1) / kRows)), dim3(kBlock), 0, st,
                         in, S, cps, reinterpret_cast<const Stats*>(stats), teacher_mass, grad_loss, temperature,
                         static_cast<T*>(grad_x));
      return check_launch(who);
    };
    constexpr int kW = kChunk<T>;
    const int nc = (V + kW - 1) / kW;
    if (wavefront_row<T>(V))
      return with_lanes<T>(V, [&](auto WC, auto LC, auto UC) { return launch(WC, LC, UC, 1, V); });
    constexpr int U = 16 / kW * 2;  // 32 values a thread
    const int S = (nc + kBlock * U - 1) / (kBlock * U);
    return launch(IC<kW>(), IC<kBlock>(), IC<U>(), S, (nc + S - 1) / S);
  });
}

}  // extern "C"

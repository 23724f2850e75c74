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
// The sums over i are over places: places that name one class count with their
// masses each, sum p_i log(P / p_i) below the term of their joined mass P, a constant
// of the logits. q_rest and the gradient's p_j are of classes.
// With A = sum p + r, the gradient of x_j is g T (A q_j - p_j) for a listed
// class and g T (A q_rest - r) q_j / q_rest for the others (r = 0, q_rest = 1
// for a renormalised list): one exponential a class, relative to the statistics
// of the classes outside the list, where A q_rest - r does not cancel in
// float32 and nothing overflows however small q_rest is.
//
// The forward reads the logits once (rowsoftmax.h); with the tail, listed
// classes are marked in a bitmap in LDS and left out of the sums, which a
// subtraction from the whole sum could not recover where the list holds nearly
// all of the mass. What remains is K values a row, which its lanes finish. log p
// - log q is a difference of near values: the logarithms, differences, products
// and sums over the list are float64, the logarithm of a float32 sum to 2^-24
// (log_of), and so are the exponentials of the tail's masses, whose sum is taken
// from one. Those of a renormalised list are float32 to 2 ulp (exp_of): an error of
// the masses, which the backward keeps in float32 as well. The backward reads
// the logits, writes the gradient of a class outside the list for every class, and
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
  float c;       // log2(e) / T
  double c_ln2;  // c ln 2
  double temperature;
  int K;
  const float* t;        // [n, K]
  const int64_t* index;  // [n, K]
};

// What the backward takes of a row.
struct Stats {
  float mb, cb;     // gradient of a class outside the list: cb 2^d, d by Shift(mb)
  float m, l2s, a;  // of a listed class: a 2^(d - l2s) - p, d by Shift(m)
  float pad[3];
};

struct Out {
  float* loss;
  Stats* stats;  // NULL: neither is kept
  float* p;      // [n, K]: the teacher's mass at the place's class, over all places that name it
};

template <int LPR>
__device__ __forceinline__ double lanes_sum(double v) {
  for_offsets<1, LPR>([&](auto OC) {
    constexpr int o = decltype(OC)::value;
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __float_as_uint(xor_shfl<o>(__uint_as_float(static_cast<uint32_t>(b))));
    const uint32_t hi = __float_as_uint(xor_shfl<o>(__uint_as_float(static_cast<uint32_t>(b >> 32))));
    v += __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
  });
  return v;
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
  for_offsets<1, LPR>([&](auto OC) { v += xor_shfl<decltype(OC)::value>(v); });
  return v;
}

template <int LPR>
__device__ __forceinline__ float lanes_max(float v) {
  for_offsets<1, LPR>([&](auto OC) { v = fmaxf(v, xor_shfl<decltype(OC)::value>(v)); });
  return v;
}

// What is known of a row's list once its lanes have been through it once.
struct ListSummary {
  float top, top_x;    // the teacher's largest value, the student's largest logit (of a listed class)
  bool any, bad;       // a place that names a class; one that names none of the V
};

// The student over all classes, from its statistics (m, s) outside the list
// (TAIL; over all classes otherwise) and the listed logits' sum.
struct Student {
  Shift rest, all;
  float s;       // relative to `rest`
  double log_s;  // of the sum over all classes, relative to the exact product m c of `all` (LogProb::base)
  bool none;     // no class left
  __device__ __forceinline__ Student(float m, float s_, float mt, float c) : rest(m, c), all(mt, c), s(s_) {}
  __device__ __forceinline__ void total(float listed) {
    const float st = listed + (s == 0.0f ? 0.0f : s * __builtin_amdgcn_exp2f(all.d_of(rest.m)));
    none = st == 0.0f;
    log_s = (none ? 0.0 : log_of(st)) + all.rounding() * kLn2d;
  }
  // (no class left: every logit is -inf, and so is log q)
  __device__ __forceinline__ LogProb log_q(double c_ln2) const { return LogProb(all.m, c_ln2, log_s); }
};

// e^v of a float64 difference v to 2 ulp of float32: what rounding v loses is
// multiplied back.
__device__ __forceinline__ double exp_of(double v) {
  const float hi = static_cast<float>(v), e = expf(hi);
  return hi == -kInf ? 0.0 : fmaf(e, static_cast<float>(v - hi), e);
}

// The row's loss and statistics from the sums over its list, by one lane.
template <typename T, bool TAIL>
__device__ __forceinline__ void conclude(const In<T>& in, const Out& o, int64_t r, const Student& q,
                                         const ListSummary& list, float members, double loss, double mass) {
  double a = mass, cb = mass;
  if constexpr (TAIL) {
    const double left = list.any && members < in.V ? fmax(0.0, 1.0 - mass) : 0.0;
    const double lrest = q.s == 0.0f ? -kInfd : (q.rest.origin() - q.all.exact()) * kLn2d + (log_of(q.s) - q.log_s);
    if (left > 0.0) {  // its logarithm: that of the nearest float32, and what the rounding left
      const float l = static_cast<float>(left);
      loss += left * (log_of(l) + static_cast<float>(left - l) / l - lrest);
    }
    a = mass + left;
    cb = a * exp_of(lrest) - left;
  }
  if (list.bad) loss = a = cb = __builtin_nan("");
  o.loss[r] = static_cast<float>(loss * in.temperature * in.temperature);
  if (o.stats)
    o.stats[r] = Stats{q.rest.m,  // (no class outside the list: 0, or NaN as it is)
                       q.s == 0.0f ? 0.0f * static_cast<float>(cb) : static_cast<float>(cb) / q.s, q.all.m,
                       q.none ? kInf : static_cast<float>(q.log_s * (1.0 / kLn2d) - q.all.rounding()),
                       static_cast<float>(a),
                       {0.0f, 0.0f, 0.0f}};
}

// e^(t - top) of a list that is renormalised. What a list leaves of one (1 - sum
// e^t, near 0 for a confident teacher) takes the exponential itself in float64.
__device__ __forceinline__ double list_exp(float t, float top) {
  return exp_of(static_cast<double>(t) - shift_of(top));
}

template <bool TAIL>
__device__ __forceinline__ double list_p(float t, float top, double inv_total) {
  if constexpr (TAIL) return exp(static_cast<double>(t));
  return list_exp(t, top) * inv_total;
}

// Row r by LPR < 64 lanes (lane q), from the joined statistics (m, s) of the
// classes outside the list (TAIL) or of all classes; `again`: a class is named
// twice. Rows this short have short lists: each lane goes through its places
// once for every step.
template <typename T, int LPR, bool TAIL>
__device__ void finish(const In<T>& in, const Out& o, int64_t r, int q, float m, float s, bool again) {
  const int64_t* index = in.index + r * in.K;
  const float* t = in.t + r * in.K;
  const T* row = in.x + r * in.ld;
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
    if (TAIL) top_x = fmaxf(top_x, to_f32(row[j]));
  }
  const ListSummary list{lanes_max<LPR>(top), lanes_max<LPR>(top_x), lanes_max<LPR>(any) != 0.0f,
                         lanes_max<LPR>(bad) != 0.0f};
  Student st(m, s, TAIL ? shift_of(fmaxf(s == 0.0f ? -kInf : m, list.top_x)) : m, in.c);
  float members = 0.0f, listed = 0.0f;
  double total = 0.0;
  for (int i = q; i < in.K; i += LPR) {
    const int64_t j = index[i];
    if (j < 0 || j >= in.V) continue;
    if constexpr (TAIL) {
      bool first = true;
      if (again)
        for (int k = 0; k < i; ++k) first = first && index[k] != j;
      if (!first) continue;
      members += 1.0f;
      listed += __builtin_amdgcn_exp2f(st.all.d(to_f32(row[j])));
    } else {
      total += list_exp(t[i], list.top);
    }
  }
  st.total(group_sum<LPR>(listed));
  members = group_sum<LPR>(members);
  total = lanes_sum<LPR>(total);
  // log p = (t - from) - norm, the difference first: a sum of both subtrahends
  // would round norm away where all places are at -3e38
  const double from = TAIL ? 0.0 : shift_of(list.top);
  const double norm = total == 0.0 ? 0.0 : log_of(static_cast<float>(total));
  const double inv = total == 0.0 ? 1.0 : 1.0 / total;
  const LogProb log_q = st.log_q(in.c_ln2);
  double loss = 0.0, mass = 0.0;
  for (int i = q; i < in.K; i += LPR) {
    const int64_t j = index[i];
    double at_class = 0.0;
    if (j >= 0 && j < in.V) {
      const double p = list_p<TAIL>(t[i], list.top, inv);
      if (p != 0.0) {
        loss += p * (static_cast<double>(t[i]) - from - norm - log_q(to_f32(row[j])));
        mass += p;
      }
      at_class = p;
      if (o.p && again) {  // in the list's order: places of one class get the same bits
        at_class = 0.0;
        for (int k = 0; k < in.K; ++k)
          if (index[k] == j) at_class += list_p<TAIL>(t[k], list.top, inv);
      }
    }
    if (o.p) o.p[r * in.K + i] = static_cast<float>(at_class);
  }
  loss = lanes_sum<LPR>(loss);
  mass = lanes_sum<LPR>(mass);
  if (q == 0) conclude<T, TAIL>(in, o, r, st, list, members, loss, mass);
}

// The same by a whole wavefront: up to two places a lane in registers, the
// list's classes and masses in the wavefront's part of LDS, where a place finds
// the others that name its class (repeats: 0 none do, 1 some, -1 not known).
constexpr int kClaims = 512;
struct alignas(16) WaveList {
  int index[kMaxList];  // -1: names no class
  float p[kMaxList];
  uint8_t claim[kClaims];
};

__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Whether two places of a wavefront's list name one class: every place claims
// the slot of its class's hash and reads who holds it now, itself, another place
// of its class, or one of another class, in which case all places of its class try
// again with another hash. Some place of every claimed slot is done in each
// round, so the rounds end; 128 different classes take two or three. (Each place
// compared with every other instead: the join of 2,048 rows of 128 places 18 us,
// with this 11.)
template <int E>
__device__ __forceinline__ bool any_repeats(const int (&at)[E], int lane, WaveList& lds) {
  bool open[E], same = false, more = false;
#pragma unroll
  for (int e = 0; e < E; ++e) more = (open[e] = at[e] >= 0) || more;
  for (uint32_t factor = 0x9e3779b1u; __any(more); factor = factor * 5 + 2 * kClaims) {
    more = false;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (open[e]) lds.claim[static_cast<uint32_t>(at[e]) * factor >> 23] = lane + e * kWave;
    wave_lds_fence();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!open[e]) continue;
      const int holder = lds.claim[static_cast<uint32_t>(at[e]) * factor >> 23];
      open[e] = lds.index[holder] != at[e];
      same = same || (!open[e] && holder != lane + e * kWave);
      more = more || open[e];
    }
    wave_lds_fence();
  }
  static_assert(kClaims == 1 << (32 - 23), "the hash's bits");
  return __any(same);
}

template <typename T, bool TAIL, int E>
__device__ __forceinline__ void finish_places(const In<T>& in, const Out& o, int64_t r, int lane, float m, float s,
                                              int repeats, WaveList& lds) {
  int at[E];
  float t[E], x[E];
  float top = -kInf, top_x = -kInf;
  bool any = false, bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + e * kWave;
    const bool in_list = i < in.K;
    const int64_t j = in_list ? in.index[r * in.K + i] : -1;
    t[e] = in_list ? in.t[r * in.K + i] : 0.0f;
    any = any || j >= 0;
    bad = bad || j >= in.V;
    at[e] = j >= 0 && j < in.V ? static_cast<int>(j) : -1;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = at[e] >= 0 ? to_f32(in.x[r * in.ld + at[e]]) : 0.0f;
  wave_lds_fence();  // the former row's list has been read
#pragma unroll
  for (int e = 0; e < E; ++e) lds.index[lane + e * kWave] = at[e];
  wave_lds_fence();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (at[e] >= 0) {
      top = fmaxf(top, t[e]);
      top_x = fmaxf(top_x, x[e]);
    }
  const ListSummary list{lanes_max<kWave>(top), lanes_max<kWave>(top_x), __any(any) != 0, __any(bad) != 0};
  // the places that name the same class, unless the caller knows of none
  bool first[E], again = false;
#pragma unroll
  for (int e = 0; e < E; ++e) first[e] = at[e] >= 0;
  if (repeats < 0 ? any_repeats<E>(at, lane, lds) : repeats != 0) {
    for (int k = 0; k < in.K; k += 4) {
      const int4 j = *reinterpret_cast<const int4*>(&lds.index[k]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = lane + e * kWave;
        const bool b0 = j.x == at[e] && k != i, b1 = j.y == at[e] && k + 1 != i;
        const bool b2 = j.z == at[e] && k + 2 != i, b3 = j.w == at[e] && k + 3 != i;
        const bool same = at[e] >= 0 && (b0 || b1 || b2 || b3);
        again = again || same;
        if (same && ((b0 && k < i) || (b1 && k + 1 < i) || (b2 && k + 2 < i) || (b3 && k + 3 < i))) first[e] = false;
      }
    }
  }
  Student st(m, s, TAIL ? shift_of(fmaxf(s == 0.0f ? -kInf : m, list.top_x)) : m, in.c);
  float members = 0.0f, listed = 0.0f;
  double total = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (at[e] < 0) continue;
    if constexpr (TAIL) {
      members += first[e] ? 1.0f : 0.0f;
      listed += first[e] ? __builtin_amdgcn_exp2f(st.all.d(x[e])) : 0.0f;
    } else {
      total += list_exp(t[e], list.top);
    }
  }
  if constexpr (TAIL) {
    listed = group_sum<kWave>(listed);
    members = group_sum<kWave>(members);
  } else {
    total = lanes_sum<kWave>(total);
  }
  st.total(listed);
  // log p = (t - from) - norm, the difference first: a sum of both subtrahends
  // would round norm away where all places are at -3e38
  const double from = TAIL ? 0.0 : shift_of(list.top);
  const double norm = total == 0.0 ? 0.0 : log_of(static_cast<float>(total));
  const double inv = total == 0.0 ? 1.0 : 1.0 / total;
  const LogProb log_q = st.log_q(in.c_ln2);
  double loss = 0.0, mass = 0.0;
  float at_class[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    at_class[e] = 0.0f;
    if (at[e] < 0) continue;
    const double p = list_p<TAIL>(t[e], list.top, inv);
    at_class[e] = static_cast<float>(p);
    if (p != 0.0) {
      loss += p * (static_cast<double>(t[e]) - from - norm - log_q(x[e]));
      mass += p;
    }
  }
  if (o.p) {
    if (__any(again)) {
#pragma unroll
      for (int e = 0; e < E; ++e) lds.p[lane + e * kWave] = at_class[e];
      wave_lds_fence();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (at[e] < 0) continue;
        double sum = 0.0;
        for (int k = 0; k < in.K; ++k) sum += lds.index[k] == at[e] ? lds.p[k] : 0.0f;
        at_class[e] = static_cast<float>(sum);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + e * kWave < in.K) o.p[r * in.K + lane + e * kWave] = at_class[e];
  }
  loss = lanes_sum<kWave>(loss);
  mass = lanes_sum<kWave>(mass);
  if (lane == 0) conclude<T, TAIL>(in, o, r, st, list, members, loss, mass);
}

template <typename T, bool TAIL>
__device__ __forceinline__ void finish_wave(const In<T>& in, const Out& o, int64_t r, int lane, float m, float s,
                                            int repeats, WaveList& lds) {
  static_assert(kMaxList == 2 * kWave, "one or two places a lane");
  if (in.K <= kWave)
    finish_places<T, TAIL, 1>(in, o, r, lane, m, s, repeats, lds);
  else
    finish_places<T, TAIL, 2>(in, o, r, lane, m, s, repeats, lds);
}

// Masks a share's chunk: the values that another chunk owns and, TAIL, the
// listed classes: the W bits of the bitmap from its place on, moved to where its
// own values are.
template <typename T, int W, bool TAIL>
__device__ __forceinline__ void mask_chunk(typename RowChunk<T, W>::Raw& raw, const uint32_t* bits, int place, int own) {
  uint32_t listed = 0;
  if constexpr (TAIL) {
    if constexpr (W == 8)
      listed = reinterpret_cast<const uint8_t*>(bits)[place];
    else
      listed = bits[place * W >> 5] >> (place * W & 31) & ((1u << W) - 1u);
  }
  if ((listed | own) != 0) mask_out<T, W>(raw, ((1u << own) - 1u) | ((listed << own) & ((1u << W) - 1u)));
}

// Rows that LPR lanes hold. The bitmap also tells whether a list names a class
// twice: a bit that was set (60,000 rows of 128 classes with whole lists: 72 us,
// 933 with every place looking for others). 24,492 x 18 float32 with 5 places
// 6.0 us, 24,492 x 1000 bf16 with 64 25 us, 28 with the tail: what they read takes
// 0.7 and 14 us, the rest is the dependent loads of the list and its logits, and
// its sums.
// Eight float32 chunks a lane are held to three wavefronts a SIMD, the tail's one
// register more than they have (24,492 x 2000 with 64 places: two 65 us, three 50).
template <typename T, int W, int LPR, int U, bool TAIL>
__global__ __launch_bounds__(kBlock, W == 4 && U == 8 ? 3 : 1) void lanes_kernel(In<T> in, Out o) {
  constexpr int kRows = kBlock / LPR;
  constexpr int kWords = (LPR * U * W + 31) / 32;
  __shared__ uint32_t bitmap[kRows * kWords];
  __shared__ int repeats[kRows];
  __shared__ WaveList lists[LPR == kWave ? kWavesPerBlock : 1];
  const int q = threadIdx.x & (LPR - 1);
  const int slot = threadIdx.x / LPR;
  uint32_t* bits = bitmap + slot * kWords;
  const int nc = (in.V + W - 1) / W;
  Share<T, W, U> sh;
  sh.place(q, LPR, nc, in.V);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < in.n; base += step) {
    const int64_t r = base + slot;
    const bool active = r < in.n;
    if (active) sh.load(in.x + r * in.ld);
    __syncthreads();  // the former rows' bits have been read
    for (int i = q; i < kWords; i += LPR) bits[i] = 0;
    if (q == 0) repeats[slot] = 0;
    __syncthreads();
    if (active)
      for (int i = q; i < in.K; i += LPR) {
        const int64_t j = in.index[r * in.K + i];
        if (j < 0 || j >= in.V) continue;
        const uint32_t bit = 1u << (j & 31);
        if (atomicOr(&bits[j >> 5], bit) & bit) repeats[slot] = 1;
      }
    __syncthreads();
    if (!active) continue;
    const int again = repeats[slot];
#pragma unroll
    for (int u = 0; u < U; ++u)
      mask_chunk<T, W, TAIL>(sh.raw[u], bits, q + u * LPR, sh.own[u]);
    float m = sh.largest(), s = 0.0f, t = 0.0f;
    sh.template sums<false>(Shift(shift_of(m), in.c), s, t);
    join<LPR, false>(m, s, t, in.c);
    if constexpr (LPR == kWave)
      finish_wave<T, TAIL>(in, o, r, q, m, s, again, lists[wave_id()]);
    else
      finish<T, LPR, TAIL>(in, o, r, q, m, s, again != 0);
  }
}

// Slices of long rows: (m, s) to part[r * S + slice]; a row's only slice finishes
// it. 2,048 x 131,072 bf16 with 128 places and the tail 85 us (537 MB at 6.3 TB/s,
// VALU 70% busy), 4,096 x 32,000 bf16 39 us (262 MB at 6.7 TB/s).
template <typename T, int U, bool TAIL, bool PAST>
__global__ __launch_bounds__(kBlock) void slice_kernel(In<T> in, Out o, Slicing sl, float2* part) {
  constexpr int W = kChunk<T>;
  constexpr int kWords = kBlock * U * W / 32;
  __shared__ float slots[2 * kWavesPerBlock][3];
  __shared__ uint32_t bits[TAIL ? kWords : 1];
  __shared__ WaveList list;
  BlockJoin across(slots);
  const int nc = (in.V + W - 1) / W;
  const int slice = blockIdx.x;
  const int64_t r = slice_row();
  if (r >= in.n) return;
  const int begin = slice * sl.cps, end = min(begin + sl.cps, nc);
  Share<T, W, U> sh;
  sh.place(begin + threadIdx.x, kBlock, end, in.V);
  sh.template load<PAST>(in.x + r * in.ld);
  if constexpr (TAIL) {
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
    mask_chunk<T, W, TAIL>(sh.raw[u], bits, threadIdx.x + u * kBlock, sh.own[u]);
  float m = sh.largest(), s = 0.0f, t = 0.0f;
  sh.template sums<false>(Shift(shift_of(m), in.c), s, t);
  join<kWave, false>(m, s, t, in.c);
  across.run<false>(m, s, t, in.c);
  if (sl.S == 1) {
    if (threadIdx.x < kWave) finish_wave<T, TAIL>(in, o, r, threadIdx.x, m, s, -1, list);
  } else if (threadIdx.x == 0) {
    part[r * sl.S + slice] = make_float2(s == 0.0f ? -kInf : m, s);
  }
}

// Rows from their slices, a wavefront a row; lane i holds slice i. 2,048 rows of
// 128 places 11 us, 301 of 17 5 us: the slices, the list, its logits and its sums
// are loads and reductions behind each other.
template <typename T, bool TAIL>
__global__ __launch_bounds__(kBlock) void join_kernel(In<T> in, Out o, int S, const float2* part) {
  __shared__ WaveList lists[kWavesPerBlock];
  const int lane = lane_id();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWavesPerBlock;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_id(); r < in.n; r += step) {
    const float2 p = lane < S ? part[r * S + lane] : make_float2(-kInf, 0.0f);
    float m = p.x, s = p.y, t = 0.0f;
    join<kWave, false>(m, s, t, in.c);
    finish_wave<T, TAIL>(in, o, r, lane, m, s, -1, lists[wave_id()]);
  }
}

// grad_x of rows held by LPR threads (lanes, or LPR = 256: the slices of a
// long row). A row without a listed class, or whose g is zero, is zeros,
// whatever its logits hold. 2,048 x 131,072 bf16: 175 us, 1.07 GB at 6.1 TB/s,
// which HBM bounds; 301 x 50,001 float32 20 us (120 MB).
template <typename T, int W, int LPR, int U, int PASS>
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
    const Shift sf(st.mb, in.c);
    const float gt = g_loss[r] * temperature;
    const bool zero = gt == 0.0f || st.a == 0.0f;
    T* row = gx + r * in.V;
    if (active) {
      Share<T, W, U> sh;
      sh.place(begin + q, LPR, end, in.V);
      if (!zero) sh.template load<PASS == kPast>(in.x + r * in.ld);
      const float cb = gt * st.cb;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[W];
        if (zero) {
#pragma unroll
          for (int w = 0; w < W; ++w) v[w] = 0.0f;
        } else {
          X::unpack(sh.raw[u], v);
          const auto turn = [&](auto of) {
#pragma unroll
            for (int w = 0; w < W; ++w) v[w] = cb * __builtin_amdgcn_exp2f(of(v[w]));
          };
          if (sf.far)
            turn([&](float x) { return sf.far_d(x); });
          else
            turn([&](float x) { return sf.near_d(x); });
        }
        Share<T, W, U>::template store<PASS != kThrough>(row, sh.at[u], sh.own[u], v);
      }
    }
    __syncthreads();  // the listed classes are written over what another thread of this workgroup stored
    if (active && !zero)
      for (int i = q; i < in.K; i += LPR) {
        const int64_t j = in.index[r * in.K + i];
        if (j < static_cast<int64_t>(begin) * W || j >= static_cast<int64_t>(end) * W || j >= in.V) continue;
        const float x = to_f32(in.x[r * in.ld + j]);
        row[j] = from_f32<T>(gt * (st.a * __builtin_amdgcn_exp2f(Shift(st.m, in.c).d(x) - st.l2s) - p[r * in.K + i]));
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
  const float c = kLog2e / temperature;
  return In<T>{n, V, static_cast<const T*>(x), ld, c, c * kLn2d, temperature, K, t, index};
}

template <typename T>
int64_t workspace_bytes(int64_t n, int V) {
  if (wavefront_row<T>(V)) return 0;
  const Slicing sl = slicing<T>(V, n);
  return sl.S == 1 ? 0 : n * sl.S * static_cast<int64_t>(sizeof(float2));
}

template <typename T, bool TAIL>
int forward(const char* who, hipStream_t st, const In<T>& in, const Out& o, void* workspace, int64_t bytes) {
  const int64_t needed = workspace_bytes<T>(in.n, in.V);
  if (bytes < needed || (needed && !workspace)) return set_error(kInvalid, "%s: workspace too small", who);
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
    const auto launch = [&](auto PC) {
      hipLaunchKernelGGL((slice_kernel<T, U, TAIL, decltype(PC)::value>), slice_grid(sl.S, in.n), dim3(kBlock), 0, st, in,
                         o, sl, part);
    };
    pass_of<T>(in.n, in.V) == kPast ? launch(std::true_type()) : launch(std::false_type());
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
      // lane groups narrower than a wavefront: rows of a few classes, never that many bytes in earnest
      with_pass(LPR < kWave ? kThrough : pass_of<T>(n, V), [&](auto PC) {
        constexpr int PASS = LPR < kWave ? kThrough : decltype(PC)::value;
        hipLaunchKernelGGL((grad_kernel<T, W, LPR, U, PASS>), dim3(grid_of((n * S + kRows - 1) / kRows)), dim3(kBlock), 0,
                           st, in, S, cps, reinterpret_cast<const Stats*>(stats), teacher_mass, grad_loss, temperature,
                           static_cast<T*>(grad_x));
      });
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

// What the operators over rows of logits share (class_logprobs.hip,
// distill.hip): how a row is laid over threads, and its softmax statistics.
//
// l = x / T is the row's logits at temperature T and c = log2(e) / T, so that
// exp(l - l_max) = 2^d with d = x c - m c and m the largest x: one fused
// multiply-add and one hardware exponential (v_exp_f32) a term. The product
// m c is rounded, the same way wherever it is formed, so its error shifts every
// term and the result's own x alike and cancels (Shift); the fused form rounds d
// alone. A row's statistics are (m, s, t):
//   s = sum 2^d, t = sum 2^d d,
// in float32; a masked class (-inf) adds nothing to either. A row of masked
// classes alone has s = 0.
//
// Rows of up to 64 lanes x 8 chunks belong to lanes of one wavefront (the
// next power of two of the row's chunks); longer rows are cut into slices, a
// workgroup each, whose statistics a second kernel joins. Either way the
// values stay in registers between the largest value and the sums, so the
// logits are read once.
#pragma once

#include "rowvec.h"

namespace cign {
namespace rowsoftmax {
using namespace rowvec;

constexpr int kMaxClasses = 1 << 20;
constexpr int kMaxList = 128;   // entries of a row's list of classes
constexpr int kMaxSlices = 64;  // one lane of the joining wavefront each
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_huge_valf();
constexpr double kLn2d = 0.6931471805599453, kInfd = __builtin_huge_val();
// Below this power of two a float32 exponential is zero: what a logarithm that
// multiplies it may be raised to, so that 0 * -inf counts nothing.
constexpr float kFloor = -256.0f;

template <int N>
using IC = std::integral_constant<int, N>;

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Value `at` of a row: a 32-bit offset, so that a row of the whole wavefront's
// keeps its address in scalar registers.
template <typename T>
__device__ __forceinline__ T* within(T* row, int at) {
  using Byte = typename std::conditional<std::is_const<T>::value, const char, char>::type;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(row) + static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(T)));
}

// Workgroups of a launch that strides over its items.
constexpr int64_t kMaxGrid = 1 << 20;
inline int grid_of(int64_t items) { return static_cast<int>(items < kMaxGrid ? items : kMaxGrid); }
// Of one with a workgroup for each of a row's S slices, which follow each other,
// and the row of a workgroup (at or past the last one: none). No loop over
// rows, out of which the compiler would take the masks of every chunk, at twice
// the registers.
constexpr int64_t kGridRows = 65535;
inline dim3 slice_grid(int S, int64_t rows) {
  return dim3(S, static_cast<uint32_t>(rows < kGridRows ? rows : kGridRows),
              static_cast<uint32_t>((rows + kGridRows - 1) / kGridRows));
}
__device__ __forceinline__ int64_t slice_row() { return blockIdx.z * kGridRows + blockIdx.y; }

// f(IC<W>, IC<LPR>, IC<U>) for rows of V values of T that a wavefront holds,
// -1 for longer ones.
template <typename T, class F>
int with_lanes(int V, F&& f) {
  constexpr int W = kChunk<T>;
  if (V < W) {
    if (V <= 1) return f(IC<1>(), IC<1>(), IC<1>());
    if (V <= 2) return f(IC<1>(), IC<2>(), IC<1>());
    if (V <= 4) return f(IC<1>(), IC<4>(), IC<1>());
    return f(IC<1>(), IC<8>(), IC<1>());
  }
  const int nc = (V + W - 1) / W;
  if (nc <= 1) return f(IC<W>(), IC<1>(), IC<1>());
  if (nc <= 2) return f(IC<W>(), IC<2>(), IC<1>());
  if (nc <= 4) return f(IC<W>(), IC<4>(), IC<1>());
  if (nc <= 8) return f(IC<W>(), IC<8>(), IC<1>());
  if (nc <= 16) return f(IC<W>(), IC<16>(), IC<1>());
  if (nc <= 32) return f(IC<W>(), IC<32>(), IC<1>());
  if (nc <= 64) return f(IC<W>(), IC<64>(), IC<1>());
  if (nc <= 128) return f(IC<W>(), IC<64>(), IC<2>());
  if (nc <= 256) return f(IC<W>(), IC<64>(), IC<4>());
  if (nc <= 512) return f(IC<W>(), IC<64>(), IC<8>());
  return -1;
}

template <typename T>
bool wavefront_row(int V) {
  return V <= 512 * kChunk<T>;
}

// The slices of long rows: S a row, of cps chunks each, U chunks a thread
// (256 U >= cps). Eight chunks a thread (128 bytes in flight: 777 x 50,001 floats
// with top classes 34 us, 53 with 16 chunks and 35 with 4; 2,048 x 131,072 bf16
// with a list 82, 86 with 4), 16 where 64 slices would not cover the row, fewer
// while that leaves fewer than 1024 workgroups, so that few rows still spread over
// the card.
struct Slicing {
  int U, S, cps;
};

// How the logits and their gradient pass the 256 MB cache behind the L2s: read
// and written through it; from 144 MiB of logits on the gradient is written past
// it, whose lines would push the logits and each other out; from 320 MiB on,
// where nothing is left for the next pass anyway, the logits are read past it too,
// both ways. Measured, forward and gradient of a list's loss: 128 MiB of bf16
// logits 75 us through, 76 with the gradient past, 80 with both past; 160 MiB 92,
// 88, 91; 256 MiB 167, 137, 137 (of float32 161, 127, 142); 384 MiB 255, 221,
// 201; 512 MiB 334, 300, 264; 1.5 GiB 941, 896, 835. Followed at once by a kernel that reads the
// gradient, 160 to 200 MB take 8% less past the cache, 268 MB and more 2 to 4%
// more.
enum Pass : int { kThrough = 0, kWritePast = 1, kPast = 2 };
inline Pass pass_of(int64_t bytes) {
  return bytes >= 320ll << 20 ? kPast : bytes >= 144ll << 20 ? kWritePast : kThrough;
}
template <typename T>
Pass pass_of(int64_t n, int V) {
  return pass_of(n * V * static_cast<int64_t>(sizeof(T)));
}
// f(IC<Pass>)
template <class F>
void with_pass(Pass p, F&& f) {
  if (p == kThrough) f(IC<kThrough>());
  else if (p == kWritePast) f(IC<kWritePast>());
  else f(IC<kPast>());
}

template <typename T>
Slicing slicing(int V, int64_t n) {
  constexpr int W = kChunk<T>;
  const int nc = (V + W - 1) / W;
  auto slices = [&](int u) { return (nc + kBlock * u - 1) / (kBlock * u); };
  int U = slices(8) <= kMaxSlices ? 8 : 16;
  while (U > 1 && n * slices(U) < 1024 && slices(U / 2) <= kMaxSlices) U /= 2;
  const int S = slices(U), cps = (nc + S - 1) / S;
  while (U > 1 && kBlock * (U / 2) >= cps) U /= 2;
  return Slicing{U, S, cps};
}

template <typename T, class F>
int with_chunks(int U, F&& f) {
  if (U <= 1) return f(IC<1>());
  if (U <= 2) return f(IC<2>());
  if (U <= 4) return f(IC<4>());
  if (U <= 8) return f(IC<8>());
  if constexpr (sizeof(T) == 4) return f(IC<16>());
  return -1;
}

// The values of a raw chunk whose bit of `kill` is set become -inf. Chunks
// that keep all of theirs (nearly every one) skip the work together.
template <typename T, int W>
__device__ __forceinline__ void mask_out(typename RowChunk<T, W>::Raw& q, uint32_t kill) {
  if (kill == 0) return;
  if constexpr (W == 1) {
    q = from_f32<T>(-kInf);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (kill >> w & 1) q[w] = -kInf;
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const uint32_t lo = static_cast<int32_t>(kill << (31 - 2 * i)) >> 31, hi = static_cast<int32_t>(kill << (30 - 2 * i)) >> 31;
      const uint32_t mask = (lo & 0xffffu) | (hi & 0xffff0000u);
      q[i] = (q[i] & ~mask) | (0xff80ff80u & mask);
    }
  }
}

// d = (x - m) log2(e) / T for the classes of a row. The rounding of m c shifts
// every d by up to 2^-24 |m c|, which must stay far from what an exponential
// overflows at: from |m c| = 10^6 on (and where m c is no finite number: rows whose
// every logit is the type's lowest, tiny temperatures) the difference is taken
// first instead.
struct Shift {
  float m, c, mc;
  bool far;
  __device__ __forceinline__ Shift(float m_, float c_) : m(m_), c(c_), mc(m_ * c_), far(is_far(m_ * c_)) {}
  static __device__ __forceinline__ bool is_far(float v) { return !(fabsf(v) < 1e6f); }
  __device__ __forceinline__ float near_d(float x) const { return fmaf(x, c, -mc); }
  __device__ __forceinline__ float far_d(float x) const { return (x - m) * c; }
  __device__ __forceinline__ float d(float x) const { return far ? far_d(x) : near_d(x); }
  // of another shift's m, relative to which sums were taken: a near shift
  // stands at its rounded product, a far one at the exact one
  __device__ __forceinline__ float d_of(float other) const {
#pragma clang fp contract(off)
    const float oc = other * c;
    const bool other_far = is_far(oc);
    if (far) return other_far ? far_d(other) : fmaf(-m, c, oc);
    return other_far ? fmaf(other, c, -mc) : oc - mc;
  }
  // Where d is taken from, for differences of two shifts that float32 may not
  // hold (at T < log2(e) two ends of the type's range lie further apart): the
  // product as rounded where near, the exact one where far.
  __device__ __forceinline__ double exact() const { return static_cast<double>(m) * c; }
  __device__ __forceinline__ double origin() const { return far ? exact() : mc; }
  __device__ __forceinline__ double rounding() const { return far ? 0.0 : mc - exact(); }
};

// A thread's share of a row: U chunks at positions first, first + stride, ...
// below `end` (chunk numbers); places past the end repeat the last chunk and
// own nothing.
template <typename T, int W, int U>
struct Share {
  using X = RowChunk<T, W>;
  typename X::Raw raw[U];
  int at[U];   // first value of the chunk
  int own[U];  // its own values start here (W: none)

  __device__ __forceinline__ void place(int first, int stride, int end, int V) {
    const int last = min(end * W, V) - W;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (first + u * stride) * W;
      at[u] = min(i, last);
      own[u] = min(i - at[u], W);
    }
  }
  template <bool PAST = false>
  __device__ __forceinline__ void load(const T* row) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (PAST)
        raw[u] = X::load_past(within(row, at[u]));
      else
        raw[u] = X::load(within(row, at[u]));
    }
  }
  __device__ __forceinline__ void mask_foreign() {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (own[u] != 0) mask_out<T, W>(raw[u], (1u << own[u]) - 1u);
  }
  // f over the packed values of chunks [U0, U1) of a bf16 row.
  template <class P, int U0, int U1, class F>
  __device__ __forceinline__ P fold(F&& f) const {
    P v = __builtin_bit_cast(P, static_cast<uint32_t>(raw[U0][0]));
#pragma unroll
    for (int u = U0; u < U1; ++u)
#pragma unroll
      for (int w = u == U0; w < W / 2; ++w) v = f(v, __builtin_bit_cast(P, static_cast<uint32_t>(raw[u][w])));
    return v;
  }
  // The largest value of chunks [U0, U1); NaN may come out as itself or be
  // passed over (the sums are NaN either way).
  template <int U0 = 0, int U1 = U>
  __device__ __forceinline__ float largest() const {
    if constexpr (sizeof(T) == 2 && W > 1) {
      // On the packed bits: the signed maximum is the largest value if any is
      // positive, the unsigned minimum if none is: half an instruction a value or
      // one, where unpacking and a float maximum take two and a half.
      const i16x2 top = fold<i16x2, U0, U1>([](i16x2 a, i16x2 b) { return __builtin_elementwise_max(a, b); });
      const short t = top.x > top.y ? top.x : top.y;
      uint32_t bits = static_cast<uint16_t>(t);
      if (t < 0) {
        const u16x2 low = fold<u16x2, U0, U1>([](u16x2 a, u16x2 b) { return __builtin_elementwise_min(a, b); });
        bits = low.x < low.y ? low.x : low.y;
      }
      return __uint_as_float(bits << 16);
    } else {
      float m = -kInf;
#pragma unroll
      for (int u = U0; u < U1; ++u) {
        float v[W];
        X::unpack(raw[u], v);
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, v[w]);
      }
      return m;
    }
  }
  // Adds the share's s (and t) relative to the shift. t needs its d raised where
  // a class is masked; wavefronts of bf16 rows without one, which half an
  // instruction a value tells, do without.
  template <bool WITH_T>
  __device__ __forceinline__ void sums(const Shift& sf, float& s, float& t) const {
    const auto near_d = [&](float x) { return sf.near_d(x); };
    if (sf.far) return add<WITH_T>([&](float x) { return sf.far_d(x); }, s, t);
    if constexpr (WITH_T && sizeof(T) == 2 && W > 1) {
      // the unsigned maximum: the lowest value, or a NaN, if any is negative
      const u16x2 low = fold<u16x2, 0, U>([](u16x2 a, u16x2 b) { return __builtin_elementwise_max(a, b); });
      const uint32_t bits = low.x > low.y ? low.x : low.y;
      if (__all(near_d(__uint_as_float(bits >= 0x8000u ? bits << 16 : 0u)) > -1e30f))
        return add<WITH_T, false>(near_d, s, t);
    }
    add<WITH_T>(near_d, s, t);
  }
  template <bool WITH_T, bool MASKED = true, class D>
  __device__ __forceinline__ void add(D&& of, float& s, float& t) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[W];
      X::unpack(raw[u], v);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float d = of(v[w]);
        const float e = __builtin_amdgcn_exp2f(d);
        s += e;
        if constexpr (WITH_T) t = fmaf(e, MASKED ? fmaxf(d, kFloor) : d, t);
      }
    }
  }
  // Stores chunk u's own values of a result.
  template <bool PAST = false>
  static __device__ __forceinline__ void store(T* row, int at, int own, const float (&v)[W]) {
    if (own == 0) {
      if constexpr (PAST)
        X::store_past(within(row, at), v);
      else
        X::store(within(row, at), v);
    } else if (own < W) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (w >= own) row[at + w] = from_f32<T>(v[w]);
    }
  }
};

// The shift of a row whose largest value is m: 0 for a row without any.
__device__ __forceinline__ float shift_of(float m) { return m == -kInf ? 0.0f : m; }

// log s of a float32 sum: the exponent apart, the hardware's base-2 logarithm
// (v_log_f32, 1 ulp) of a value in [0.7, 1.42), at most 0.5, and float64 for the
// rest: below 2^-24 off. A float32 logarithm of the whole is off by half a step of
// itself, 2^-21 for s = 50,001, more than the sum that it is taken of. Lists of
// 24,492 x 100 with 64 places: 19.7 us, 20.7 with logf of the same value; float64
// functions cost 24,492 x 18 with 5 places 1.8 us more, x 1000 with 64 17.
__device__ __forceinline__ double log_of(float s) {
  float f = __builtin_amdgcn_frexp_mantf(s);
  int e = __builtin_amdgcn_frexp_expf(s);
  if (f < 0.70710678f) {
    f += f;
    --e;
  }
  return (e + static_cast<double>(__builtin_amdgcn_logf(f))) * kLn2d;
}

// log p of a row's logits in float64: (x - m) c ln 2 - base, the difference of
// logits first, since their products with c may be far larger; base is log s and
// what the shift's product was rounded by, times ln 2.
struct LogProb {
  float m;
  double c, base;  // c ln 2 (of the whole launch: scalar registers)
  __device__ __forceinline__ LogProb(float m_, double c_ln2, double base_) : m(m_), c(c_ln2), base(base_) {}
  __device__ __forceinline__ LogProb(const Shift& sf, double c_ln2, double log_s)
      : LogProb(sf.m, c_ln2, log_s + sf.rounding() * kLn2d) {}
  __device__ __forceinline__ double operator()(float x) const { return fma(static_cast<double>(x) - m, c, -base); }
};

// Joins statistics over the LPR lanes of a group (one (m, s, t) a lane; m as
// largest() gave it, s and t relative to shift_of(m)). m becomes the shift.
// Every lane gets the same bits: a lane that contracted its own product into
// the first addition would round differently from its partner.
template <int LPR, bool WITH_T>
__device__ __forceinline__ void join(float& m, float& s, float& t, float c) {
#pragma clang fp contract(off)
  float top = m;
  for_offsets<1, LPR>([&](auto OC) { top = fmaxf(top, xor_shfl<decltype(OC)::value>(top)); });
  top = shift_of(top);
  const float d = Shift(top, c).d_of(shift_of(m));
  const float e = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(d);
  if constexpr (WITH_T) t = s == 0.0f ? 0.0f : e * fmaf(s, fmaxf(d, kFloor), t);
  s *= e;
  for_offsets<1, LPR>([&](auto OC) {
    constexpr int o = decltype(OC)::value;
    s += xor_shfl<o>(s);
    if constexpr (WITH_T) t += xor_shfl<o>(t);
  });
  m = top;
}

// The same over a workgroup of kBlock threads whose wavefronts have joined
// theirs: every thread gets the result. The slots alternate (GroupReduce), so
// this is the call's only barrier.
struct BlockJoin {
  float (*slots)[3];  // [2 * kWavesPerBlock]
  int turn = 0;
  __device__ explicit BlockJoin(float (*p)[3]) : slots(p) {}

  template <bool WITH_T>
  __device__ __forceinline__ void run(float& m, float& s, float& t, float c) {
    static_assert(kWavesPerBlock == 4, "one quad joins the wavefronts");
    float(*p)[3] = slots + turn * kWavesPerBlock;
    turn ^= 1;
    if (lane_id() == 0) {
      p[wave_id()][0] = s == 0.0f ? -kInf : m;
      p[wave_id()][1] = s;
      if constexpr (WITH_T) p[wave_id()][2] = t;
    }
    __syncthreads();
    const int k = lane_id() & 3;
    m = p[k][0];
    s = p[k][1];
    if constexpr (WITH_T) t = p[k][2];
    join<4, WITH_T>(m, s, t, c);  // the same in every quad
  }
};

}  // namespace rowsoftmax
}  // namespace cign

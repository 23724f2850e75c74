// Log probabilities of given classes, entropy and the top classes of rows of
// logits, and the gradient of the first two.
//
// With l = x / T, lse = log sum e^l and p = e^(l - lse):
//   logprob = l[label] - lse, entropy = -sum p (l - lse) = ln2 (log2 s - t / s)
//   (m, s, t: rowsoftmax.h), top classes by x, the lowest index first among
//   equals;
//   grad_x[j] = (g ([j = label] - p_j) - h p_j (log p_j + entropy)) / T for the
//   gradients g of logprob and h of entropy.
// The forward reads the logits once, the backward reads them once and writes
// their gradient; nothing of the row's length is kept between the two, only
// (m, log2 s, entropy) of each row.
//
// Top classes are ordered by a 64-bit key, the value's order-preserving bits
// above the complement of the index, so that every key of a row is different
// and the order never depends on which thread finds a class.
#include "rowsoftmax.h"

namespace cign {
namespace class_logprobs {
using namespace rowsoftmax;

constexpr int kCandidates = 1024;    // keys a slice's selection keeps in LDS
constexpr int kShortTopRow = 512;    // longest row whose top classes lane groups pick

// NaN counts as -inf, -0 as +0.
__device__ __forceinline__ float ranked(float x) { return fmaxf(x, -kInf) + 0.0f; }
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t b = __float_as_uint(ranked(x));
  const uint32_t u = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(u) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
// The value of a key, -inf for the bar below every key.
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return u == 0 ? -kInf : __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }

// A row's outputs, written by one thread.
struct Out {
  const int64_t* label;  // NULL: none asked for
  int64_t ignore;
  float* logprob;
  float* entropy;
  float* stats;  // [n, 4]: m, log2 s (inf: no class left), entropy, 1 / s; NULL: not kept
  int K;
  float* top_logprob;
  int64_t* top_index;
};

template <typename T>
struct In {
  int64_t n;
  int V;
  const T* x;
  int64_t ld;
  float c, inv_t;  // log2(e) / T, 1 / T
  double c_ln2;    // c ln 2
};

// log p and the entropy are float64 differences of values that may be much larger,
// rounded once. A row without a class has log s = 0, so that -inf comes out.
__device__ __forceinline__ double log_sum(float s) { return s == 0.0f ? 0.0 : log_of(s); }
template <typename T>
__device__ __forceinline__ LogProb log_prob(const In<T>& in, float m, double log_s) {
  return LogProb(Shift(m, in.c), in.c_ln2, log_s);
}

// Label, entropy and statistics of row r from its joined (m, s, t) and log s.
template <typename T>
__device__ __forceinline__ void finish(const In<T>& in, const Out& o, int64_t r, float m, float s, float t,
                                       double log_s, const LogProb& log_p) {
  const bool none = s == 0.0f;
  // t / s: a float32 reciprocal and one step in float64
  const double inv = __builtin_amdgcn_rcpf(s), first = t * inv;
  const double mean = fma(fma(-first, static_cast<double>(s), static_cast<double>(t)), inv, first);
  const float H = none ? 0.0f : static_cast<float>(log_s - kLn2d * mean);
  o.entropy[r] = H;
  if (o.label) {
    const int64_t y = o.label[r];
    float lp = 0.0f;
    if (y != o.ignore)
      lp = y >= 0 && y < in.V ? static_cast<float>(log_p(to_f32(in.x[r * in.ld + y]))) : __builtin_nanf("");
    o.logprob[r] = lp;
  }
  if (o.stats) {
    float* p = o.stats + 4 * r;
    p[0] = m;
    p[1] = none ? kInf : static_cast<float>(log_s * (1.0 / kLn2d));
    p[2] = H;
    p[3] = static_cast<float>(inv * fma(-inv, static_cast<double>(s), 2.0));
  }
}

template <typename T>
__device__ __forceinline__ void put_top(const In<T>& in, const Out& o, int64_t r, int rank, uint64_t key,
                                        const LogProb& log_p) {
  const int i = key_index(key);
  o.top_index[r * o.K + rank] = i;
  o.top_logprob[r * o.K + rank] = static_cast<float>(log_p(to_f32(in.x[r * in.ld + i])));
}

// The largest key below `below` of a share's own values.
template <typename T, int W, int U>
__device__ __forceinline__ uint64_t best_below(const Share<T, W, U>& sh, uint64_t below) {
  uint64_t best = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[W];
    RowChunk<T, W>::unpack(sh.raw[u], v);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint64_t k = key_of(v[w], sh.at[u] + w);
      if (w >= sh.own[u] && k < below && k > best) best = k;
    }
  }
  return best;
}

// f(IC<0>) ... f(IC<N - 1>)
template <int N, int I = 0, class F>
__device__ __forceinline__ void for_each(F&& f) {
  if constexpr (I < N) {
    f(IC<I>());
    for_each<N, I + 1>(f);
  }
}

// The key of the share's largest value m, of those of its chunks: best_below(~0)
// without making every value's key, the first own value equal to m of the first
// chunk that has one. A share whose m is -inf, or with a chunk whose NaN hides
// its other values, takes the long way.
template <typename T, int W, int U>
__device__ __forceinline__ uint64_t best_key(const Share<T, W, U>& sh, const float (&of_chunk)[U], float m) {
  bool hidden = !(m > -kInf);
#pragma unroll
  for (int u = 0; u < U; ++u) hidden = hidden || of_chunk[u] != of_chunk[u];
  if (hidden) return best_below(sh, ~0ull);
  auto raw = sh.raw[0];
  int at = sh.at[0];
#pragma unroll
  for (int u = U - 1; u > 0; --u) {
    const bool here = of_chunk[u] == m;
    raw = here ? sh.raw[u] : raw;
    at = here ? sh.at[u] : at;
  }
  const bool first = of_chunk[0] == m;
  raw = first ? sh.raw[0] : raw;
  at = first ? sh.at[0] : at;
  float v[W];
  RowChunk<T, W>::unpack(raw, v);
  int index = 0;
#pragma unroll
  for (int w = W - 1; w >= 0; --w) index = v[w] == m ? at + w : index;
  return key_of(m, index);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto step = [&](auto CTRL) {
    const uint32_t o = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(CTRL)::value, 0xF, 0xF, true);
    v = o > v ? o : v;
  };
  step(IC<0xB1>());   // quad_perm [1,0,3,2]
  step(IC<0x4E>());   // quad_perm [2,3,0,1]
  step(IC<0x141>());  // row_half_mirror: the other quad of 8 (quads are uniform by now)
  step(IC<0x128>());  // row_ror:8
  step(IC<0x142>());  // row_bcast:15, a row's result to the next row
  step(IC<0x143>());  // row_bcast:31, rows 0 and 1 to rows 2 and 3
  return __builtin_amdgcn_readlane(v, kWave - 1);
}

// The largest key of LPR lanes, on all of them.
template <int LPR>
__device__ __forceinline__ uint64_t group_max(uint64_t k) {
  if constexpr (LPR == kWave) {
    const uint32_t hi = wave_max(static_cast<uint32_t>(k >> 32));
    const uint32_t lo = wave_max(static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
    return static_cast<uint64_t>(hi) << 32 | lo;
  }
  for_offsets<1, LPR>([&](auto OC) {
    constexpr int o = decltype(OC)::value;
    const uint32_t lo = __float_as_uint(xor_shfl<o>(__uint_as_float(static_cast<uint32_t>(k))));
    const uint32_t hi = __float_as_uint(xor_shfl<o>(__uint_as_float(static_cast<uint32_t>(k >> 32))));
    const uint64_t other = static_cast<uint64_t>(hi) << 32 | lo;
    if (other > k) k = other;
  });
  return k;
}

// How many of n keys in LDS (padded with zeros to a multiple of 16) are above
// `key`: every thread of the workgroup reads the same ones, eight 16-byte reads
// in flight.
__device__ __forceinline__ int count_above(const uint64_t* keys, int n, uint64_t key) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  int above = 0;
  for (int i = 0; i < n; i += 16) {
    u64x2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const u64x2*>(keys + i + 2 * k);
#pragma unroll
    for (int k = 0; k < 8; ++k) above += (v[k].x > key) + (v[k].y > key);
  }
  return above;
}

// Rows that LPR lanes hold: 24,492 x 5 float32 3.2 us (0.5 MB: a launch, the
// loads' latency and the reductions).
template <typename T, int W, int LPR, int U, bool TOP>
__global__ __launch_bounds__(kBlock) void lanes_kernel(In<T> in, Out o) {
  constexpr int kRows = kBlock / LPR;
  const int q = threadIdx.x & (LPR - 1);
  const int nc = (in.V + W - 1) / W;
  Share<T, W, U> sh;
  sh.place(q, LPR, nc, in.V);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / LPR; r < in.n; r += step) {
    sh.load(in.x + r * in.ld);
    sh.mask_foreign();
    float m = sh.largest(), s = 0.0f, t = 0.0f;
    sh.template sums<true>(Shift(shift_of(m), in.c), s, t);
    join<LPR, true>(m, s, t, in.c);
    const double log_s = log_sum(s);
    const LogProb log_p = log_prob(in, m, log_s);
    if (q == 0) finish(in, o, r, m, s, t, log_s, log_p);
    if constexpr (TOP) {
      uint64_t mine = best_below(sh, ~0ull);
      for (int k = 0; k < o.K; ++k) {
        const uint64_t best = group_max<LPR>(mine);
        if (mine == best) {  // one lane: keys differ
          put_top(in, o, r, k, best, log_p);
          mine = best_below(sh, best);
        }
      }
    }
  }
}

// Slices of long rows: (m, s, t) to part[(r * S + slice)] (a float4), the K
// largest keys, in falling order, to keys[(r * S + slice) * K ...] (0: the
// slice has no more). With S = 1 the row's outputs are written at once.
//
// Measured: 8,192 x 32,000 bf16 82 to 101 us (524 MB at 5.2 to 6.4 TB/s; the
// VALU is 78% busy with 8.5 instructions and a quarter-rate exponential a value,
// so the clock decides); 777 x 50,001 float32 with 5 top classes 34 us (155 MB at
// 4.6 TB/s; the selection's LDS rounds); one row of 131,072 bf16 with 20 over 64
// workgroups 6 us (latency).
template <typename T, int U, bool TOP, bool PAST>
__global__ __launch_bounds__(kBlock) void slice_kernel(In<T> in, Out o, Slicing sl, float4* part, uint64_t* keys) {
  constexpr int W = kChunk<T>;
  __shared__ float slots[2 * kWavesPerBlock][3];
  __shared__ __align__(16) uint64_t sample[TOP ? kBlock : 1];
  __shared__ __align__(16) uint64_t cand[TOP ? kCandidates : 1];
  __shared__ uint64_t threshold;
  __shared__ int found;
  const int nc = (in.V + W - 1) / W;
  const int lane = lane_id(), slice = blockIdx.x;
  const int64_t r = slice_row();
  if (r >= in.n) return;
  BlockJoin across(slots);
  const int64_t item = r * sl.S + slice;
  const int end = min((slice + 1) * sl.cps, nc);
  Share<T, W, U> sh;
  sh.place(slice * sl.cps + threadIdx.x, kBlock, end, in.V);
  sh.template load<PAST>(in.x + r * in.ld);
  sh.mask_foreign();
  float of_chunk[TOP ? U : 1], m = -kInf, s = 0.0f, t = 0.0f;
  if constexpr (TOP) {
    for_each<U>([&](auto UC) {
      constexpr int u = decltype(UC)::value;
      of_chunk[u] = sh.template largest<u, u + 1>();
      m = fmaxf(m, of_chunk[u]);
    });
  } else {
    m = sh.largest();
  }
  const float top = m;
  sh.template sums<true>(Shift(shift_of(m), in.c), s, t);
  join<kWave, true>(m, s, t, in.c);
  if (TOP && threadIdx.x == 0) {
    threshold = 1;
    found = 0;
  }
  uint64_t mine = 0;
  const bool quads = TOP && o.K <= kBlock / 8;
  if constexpr (TOP) {
    mine = best_key(sh, of_chunk, top);
    uint64_t best = mine;
    if (quads) {
      best = group_max<4>(mine);
      if ((threadIdx.x & 3) == 0) sample[threadIdx.x >> 2] = best;
    } else {
      sample[threadIdx.x] = best;
    }
  }
  across.run<true>(m, s, t, in.c);
  if (threadIdx.x == 0) {
    if (sl.S == 1) {
      const double log_s = log_sum(s);
      finish(in, o, r, m, s, t, log_s, log_prob(in, m, log_s));
    } else {
      part[item] = make_float4(s == 0.0f ? -kInf : m, s, t, 0.0f);
    }
  }
  if constexpr (TOP) {
    // The K-th largest of the best keys of quads (K <= 32) or threads bounds
    // the slice's K-th key from below; every key at or above it is a
    // candidate. Each quad counts the keys above its own, a quarter a lane.
    const int K = o.K;
    if (quads) {
      const uint64_t own = sample[threadIdx.x >> 2];
      int above = count_above(sample + (threadIdx.x & 3) * (kBlock / 16), kBlock / 16, own);
      above += __float_as_int(xor_shfl<1>(__int_as_float(above)));
      above += __float_as_int(xor_shfl<2>(__int_as_float(above)));
      if (own != 0 && above == K - 1) threshold = own;  // one quad: keys differ
    } else {
      const int above = count_above(sample, kBlock, mine);
      if (mine != 0 && above == K - 1) threshold = mine;
    }
    __syncthreads();
    const uint64_t bar = threshold;
    if (mine >= bar) {
      const float low = key_value(bar);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // (a chunk of NaN is looked at; on 4 values the test costs what it saves)
        if (W == 8 && of_chunk[u] < low) continue;
        float v[W];
        RowChunk<T, W>::unpack(sh.raw[u], v);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (!(ranked(v[w]) >= low)) continue;
          const uint64_t k = key_of(v[w], sh.at[u] + w);
          if (w >= sh.own[u] && k >= bar) {
            const int at = atomicAdd(&found, 1);
            if (at < kCandidates) cand[at] = k;
          }
        }
      }
    }
    __syncthreads();
    const int count = found;
    uint64_t* list = keys + item * K;
    if (count <= kCandidates) {
      for (int i = count + threadIdx.x; i < ((count + 15) & ~15); i += kBlock) cand[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < count; i += kBlock) {
        const uint64_t k = cand[i];
        const int rank = count_above(cand, count, k);
        if (rank < K) {
          if (sl.S == 1)
            put_top(in, o, r, rank, k, log_prob(in, m, log_sum(s)));
          else
            list[rank] = k;
        }
      }
      if (sl.S > 1)
        for (int i = count + threadIdx.x; i < K; i += kBlock) list[i] = 0;
    } else {
      // More candidates than the buffer holds (many large values in few
      // threads' chunks): K rounds over the registers.
      uint64_t below = ~0ull;
      for (int k = 0; k < K; ++k) {
        const uint64_t w = group_max<kWave>(best_below(sh, below));
        __syncthreads();
        if (lane == 0) sample[wave_id()] = w;
        __syncthreads();
        uint64_t best = sample[0];
        for (int i = 1; i < kWavesPerBlock; ++i) best = sample[i] > best ? sample[i] : best;
        if (threadIdx.x == 0) {
          if (sl.S == 1)
            put_top(in, o, r, k, best, log_prob(in, m, log_sum(s)));
          else
            list[k] = best;
        }
        below = best;
      }
    }
  }
}

// Rows from their slices, without top classes: a wavefront a row, lane i holds
// slice i. 8,192 rows of 2 slices 5 us, the latency of the slices' and then the
// label's load.
template <typename T>
__global__ __launch_bounds__(kBlock) void join_kernel(In<T> in, Out o, int S, const float4* part) {
  const int lane = lane_id();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWavesPerBlock;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_id(); r < in.n; r += step) {
    const float4 p = lane < S ? part[r * S + lane] : make_float4(-kInf, 0.0f, 0.0f, 0.0f);
    float m = p.x, s = p.y, t = p.z;
    join<kWave, true>(m, s, t, in.c);
    const double log_s = log_sum(s);
    if (lane == 0) finish(in, o, r, m, s, t, log_s, log_prob(in, m, log_s));
  }
}

// With top classes, a workgroup a row: of the slices' falling lists, the K-th
// largest among the first ceil(K / S) of each bounds the row's K-th key from
// below, and the keys at or above it are ranked against each other (one row of
// 131,072 with K = 20: 4 us, 10.6 by rounds of the lists' heads against each
// other; 777 rows of 7 slices with K = 5: 5 us). Lists whose candidates overflow, such as the slices of a sorted row,
// are merged by those rounds.
constexpr int kHeldKeys = 8;  // list keys a thread reads ahead

template <typename T>
__global__ __launch_bounds__(kBlock) void join_top_kernel(In<T> in, Out o, int S, const float4* part,
                                                          const uint64_t* keys) {
  __shared__ __align__(16) uint64_t sample[kBlock];
  __shared__ __align__(16) uint64_t cand[kCandidates];
  __shared__ uint64_t threshold;
  __shared__ int found;
  const int lane = lane_id(), K = o.K, total = S * K;
  const int heads = (K + S - 1) / S, list = threadIdx.x / heads;  // S heads <= K + S - 1 < kBlock
  for (int64_t r = blockIdx.x; r < in.n; r += gridDim.x) {
    const float4 p = lane < S ? part[r * S + lane] : make_float4(-kInf, 0.0f, 0.0f, 0.0f);
    const uint64_t* lists = keys + r * total;  // [S][K]
    const uint64_t mine = list < S ? lists[list * K + threadIdx.x - list * heads] : 0;
    uint64_t held[kHeldKeys];
#pragma unroll
    for (int i = 0; i < kHeldKeys; ++i) held[i] = lists[min(static_cast<int>(threadIdx.x) + i * kBlock, total - 1)];
    float m = p.x, s = p.y, t = p.z;
    __syncthreads();  // the former row's candidates have been read
    sample[threadIdx.x] = mine;
    if (threadIdx.x == 0) {
      threshold = 1;
      found = 0;
    }
    join<kWave, true>(m, s, t, in.c);
    const double log_s = log_sum(s);
    const LogProb log_p = log_prob(in, m, log_s);
    __syncthreads();
    if (mine != 0 && count_above(sample, S * heads, mine) == K - 1) threshold = mine;
    __syncthreads();
    const uint64_t bar = threshold;
    const auto offer = [&](uint64_t k) {
      if (k < bar) return;
      const int at = atomicAdd(&found, 1);
      if (at < kCandidates) cand[at] = k;
    };
#pragma unroll
    for (int i = 0; i < kHeldKeys; ++i)
      if (static_cast<int>(threadIdx.x) + i * kBlock < total) offer(held[i]);
    for (int i = threadIdx.x + kHeldKeys * kBlock; i < total; i += kBlock) offer(lists[i]);
    __syncthreads();
    const int count = found;
    if (count <= kCandidates) {
      for (int i = count + threadIdx.x; i < ((count + 15) & ~15); i += kBlock) cand[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < count; i += kBlock) {
        const uint64_t k = cand[i];
        const int rank = count_above(cand, count, k);
        if (rank < K) put_top(in, o, r, rank, k, log_p);
      }
    } else if (threadIdx.x < kWave) {
      int next = 1;
      uint64_t head = lane < S ? lists[lane * K] : 0;
      for (int k = 0; k < K; ++k) {
        const uint64_t best = group_max<kWave>(head);
        if (head == best) {  // one lane: keys differ
          put_top(in, o, r, k, best, log_p);
          head = next < K ? lists[lane * K + next] : 0;
          ++next;
        }
      }
    }
    if (threadIdx.x == kBlock - 1) finish(in, o, r, m, s, t, log_s, log_p);
  }
}

// grad_x of rows held by LPR threads (lanes, or LPR = 256: the slices of a
// long row). Rows whose gradients are both zero (an ignored label) are zeros,
// whatever their logits hold. 8,192 x 32,000 bf16: 167 us, 1.05 GB at 6.3 TB/s,
// which HBM bounds.
template <typename T, int W, int LPR, int U, bool ENT, int PASS>
__global__ __launch_bounds__(kBlock) void grad_kernel(In<T> in, int S, int cps, const int64_t* label, int64_t ignore,
                                                      const float* stats, const float* g_lp, const float* g_ent,
                                                      T* gx) {
  using X = RowChunk<T, W>;
  constexpr int kRows = kBlock / LPR;
  const int q = threadIdx.x & (LPR - 1);
  const int nc = (in.V + W - 1) / W;
  const int64_t items = in.n * S;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / LPR; item < items; item += step) {
    const int64_t r = S == 1 ? item : item / S;
    const int slice = S == 1 ? 0 : static_cast<int>(item - r * S);
    const float m = stats[4 * r], l2s = stats[4 * r + 1];
    const int64_t y = label ? label[r] : ignore;
    float g = 0.0f, h = 0.0f;
    if (g_lp && y != ignore) g = y >= 0 && y < in.V ? g_lp[r] : __builtin_nanf("");
    if (ENT) h = g_ent[r];
    if (l2s == kInf) g = h = 0.0f;  // no class left
    // 2^d (a + b log2 p_j), p_j = 2^d / s (2^(d - log2 s) would round the exponent
    // once more), and g at the label
    const float inv_s = stats[4 * r + 3] * in.inv_t;
    const float a = -(g + h * stats[4 * r + 2]) * inv_s, b = -h * kLn2 * inv_s;
    const float gl = g * in.inv_t;
    const bool zero = g == 0.0f && h == 0.0f;
    const Shift sf(m, in.c);
    Share<T, W, U> sh;
    sh.place(slice * cps + q, LPR, min((slice + 1) * cps, nc), in.V);
    if (!zero) sh.template load<PASS == kPast>(in.x + r * in.ld);
    T* row = gx + r * in.V;
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
          for (int w = 0; w < W; ++w) {
            const float d = of(v[w]);
            const float e = __builtin_amdgcn_exp2f(d);
            v[w] = e * (ENT ? fmaf(b, fmaxf(d - l2s, kFloor), a) : a);
          }
        };
        if (sf.far)
          turn([&](float x) { return sf.far_d(x); });
        else
          turn([&](float x) { return sf.near_d(x); });
        const int64_t at = y - sh.at[u];
        if (at >= 0 && at < W)
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (w == at) v[w] += gl;
      }
      Share<T, W, U>::template store<PASS != kThrough>(row, sh.at[u], sh.own[u], v);
    }
  }
}

int check_args(const char* who, int dtype, int64_t n, int V, int64_t ld, float temperature) {
  if (dtype != kF32 && dtype != kBF16) return set_error(kInvalid, "%s: dtype must be 0 or 1", who);
  if (n < 0) return set_error(kInvalid, "%s: negative row count", who);
  if (V < 1 || V > kMaxClasses) return set_error(kInvalid, "%s: requires 1<=V<=%d, got %d", who, kMaxClasses, V);
  if (ld < 0) return set_error(kInvalid, "%s: negative row stride", who);
  if (!(temperature > 0.0f && temperature < kInf)) return set_error(kInvalid, "%s: temperature must be positive", who);
  return kOk;
}

template <typename T>
In<T> input(int64_t n, int V, const void* x, int64_t ld, float temperature) {
  const float c = kLog2e / temperature;
  return In<T>{n, V, static_cast<const T*>(x), ld, c, 1.0f / temperature, c * kLn2d};
}

// Whether slices take the row: longer than a wavefront holds, or than its
// lanes' rounds pick top classes from.
template <typename T>
bool sliced(int V, int K) {
  return !wavefront_row<T>(V) || (K > 0 && V > kShortTopRow);
}

template <typename F>
int with_type(int dtype, F&& f) {
  return dtype == kF32 ? f(float()) : f(bf16());
}

template <typename T>
int64_t workspace_bytes(int64_t n, int V, int K) {
  if (!sliced<T>(V, K)) return 0;
  const Slicing sl = slicing<T>(V, n);
  return sl.S == 1 ? 0 : n * sl.S * (static_cast<int64_t>(sizeof(float4)) + 8 * K);
}

template <typename T>
int forward(const char* who, hipStream_t st, const In<T>& in, const Out& o, void* workspace, int64_t bytes) {
  const int64_t needed = workspace_bytes<T>(in.n, in.V, o.K);
  if (bytes < needed || (needed && !workspace)) return set_error(kInvalid, "%s: workspace too small", who);
  if (!sliced<T>(in.V, o.K))
    return with_lanes<T>(in.V, [&](auto WC, auto LC, auto UC) {
      constexpr int W = decltype(WC)::value, LPR = decltype(LC)::value, U = decltype(UC)::value;
      constexpr int kRows = kBlock / LPR;
      const int grid = grid_of((in.n + kRows - 1) / kRows);
      if (o.K > 0) {
        if constexpr (W * LPR * U <= kShortTopRow)
          hipLaunchKernelGGL((lanes_kernel<T, W, LPR, U, true>), dim3(grid), dim3(kBlock), 0, st, in, o);
      } else {
        hipLaunchKernelGGL((lanes_kernel<T, W, LPR, U, false>), dim3(grid), dim3(kBlock), 0, st, in, o);
      }
      return check_launch(who);
    });
  const Slicing sl = slicing<T>(in.V, in.n);
  float4* part = static_cast<float4*>(workspace);
  uint64_t* keys = reinterpret_cast<uint64_t*>(part + (sl.S == 1 ? 0 : in.n * sl.S));
  const int rc = with_chunks<T>(sl.U, [&](auto UC) {
    constexpr int U = decltype(UC)::value;
    const auto launch = [&](auto TC, auto SC) {
      hipLaunchKernelGGL((slice_kernel<T, U, decltype(TC)::value, decltype(SC)::value>), slice_grid(sl.S, in.n),
                         dim3(kBlock), 0, st, in, o, sl, part, keys);
    };
    const bool past = pass_of<T>(in.n, in.V) == kPast;
    if (o.K > 0)
      past ? launch(std::true_type(), std::true_type()) : launch(std::true_type(), std::false_type());
    else
      past ? launch(std::false_type(), std::true_type()) : launch(std::false_type(), std::false_type());
    return check_launch(who);
  });
  if (rc || sl.S == 1) return rc;
  if (o.K > 0)
    hipLaunchKernelGGL((join_top_kernel<T>), dim3(grid_of(in.n)), dim3(kBlock), 0, st, in, o, sl.S, part, keys);
  else
    hipLaunchKernelGGL((join_kernel<T>), dim3(grid_of((in.n + kWavesPerBlock - 1) / kWavesPerBlock)), dim3(kBlock), 0, st,
                       in, o, sl.S, part);
  return check_launch(who);
}

}  // namespace class_logprobs
}  // namespace cign

using namespace cign;
using namespace cign::class_logprobs;

extern "C" {

int64_t cign_class_logprobs_workspace_bytes(int32_t dtype, int64_t n, int32_t V, int32_t top_k) {
  if (n < 1 || V < 1 || V > kMaxClasses || top_k < 0 || top_k > kMaxList) return 0;
  return with_type(dtype, [&](auto t) { return workspace_bytes<decltype(t)>(n, V, top_k); });
}

int cign_class_logprobs_fwd(void* stream, int32_t dtype, int64_t n, int32_t V, const void* x, int64_t x_stride,
                            float temperature, const int64_t* label, int64_t ignore_index, int32_t top_k,
                            float* logprob, float* entropy, float* top_logprob, int64_t* top_index, float* stats,
                            void* workspace, int64_t workspace_bytes) {
  const char* who = "cign_class_logprobs_fwd";
  const int rc = check_args(who, dtype, n, V, x_stride, temperature);
  if (rc) return rc;
  if (top_k < 0 || top_k > kMaxList || top_k > V)
    return set_error(kInvalid, "%s: requires 0<=top_k<=min(V, %d), got %d", who, kMaxList, top_k);
  if (n == 0) return kOk;
  if (!x || !entropy || (label && !logprob) || (top_k > 0 && (!top_logprob || !top_index)))
    return set_error(kInvalid, "%s: null argument", who);
  const Out o{label, ignore_index, logprob, entropy, stats, top_k, top_logprob, top_index};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const In<T> in = input<T>(n, V, x, x_stride, temperature);
    return forward(who, static_cast<hipStream_t>(stream), in, o, workspace, workspace_bytes);
  });
}

int cign_class_logprobs_bwd(void* stream, int32_t dtype, int64_t n, int32_t V, const void* x, int64_t x_stride,
                            float temperature, const int64_t* label, int64_t ignore_index, const float* stats,
                            const float* grad_logprob, const float* grad_entropy, void* grad_x) {
  const char* who = "cign_class_logprobs_bwd";
  const int rc = check_args(who, dtype, n, V, x_stride, temperature);
  if (rc) return rc;
  if (n == 0) return kOk;
  if (!x || !stats || !grad_x || (grad_logprob && !label)) return set_error(kInvalid, "%s: null argument", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const In<T> in = input<T>(n, V, x, x_stride, temperature);
    const auto launch = [&](auto WC, auto LC, auto UC, int S, int cps) {
      constexpr int W = decltype(WC)::value, LPR = decltype(LC)::value, U = decltype(UC)::value;
      constexpr int kRows = kBlock / LPR;
      const int grid = grid_of((n * S + kRows - 1) / kRows);
      // lane groups narrower than a wavefront: rows of a few classes, never that many bytes in earnest
      with_pass(LPR < kWave ? kThrough : pass_of<T>(n, V), [&](auto PC) {
        constexpr int PASS = LPR < kWave ? kThrough : decltype(PC)::value;
        if (grad_entropy)
          hipLaunchKernelGGL((grad_kernel<T, W, LPR, U, true, PASS>), dim3(grid), dim3(kBlock), 0, st, in, S, cps, label,
                             ignore_index, stats, grad_logprob, grad_entropy, static_cast<T*>(grad_x));
        else
          hipLaunchKernelGGL((grad_kernel<T, W, LPR, U, false, PASS>), dim3(grid), dim3(kBlock), 0, st, in, S, cps,
                             label, ignore_index, stats, grad_logprob, grad_entropy, static_cast<T*>(grad_x));
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

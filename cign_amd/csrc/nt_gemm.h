// Products of two bf16 matrices, C[b][a] = sum_k A[a][k] B[b][k], whose rows run along
// the summed axis or (turned) across it: float32 sums, a 256 x 256 tile of C a workgroup of
// eight wavefronts, 128 rows of A by 64 of B each: 32 results of 16 x 16 in 128
// registers, v_mfma_f32_16x16x32_bf16 (16 cycles).
//
// Steps of 64 values go to LDS without passing registers (16-byte direct loads, rows
// of 128 bytes an eight lanes), into a ring of five units of 32 KB, 64 values of 256
// rows of one operand each: the two in use, the other operand's next, and the two
// after. A wavefront reads half a step's fragments (12 ds_read_b128), then multiplies
// (32 MFMAs, 512 cycles), with a barrier after each; the wavefronts 4 to 7, one on
// each SIMD beside one of 0 to 3, run one barrier behind, so that a SIMD's matrix
// unit works for one of its two wavefronts while the other reads. A row's 16-byte
// chunk c lies at place c ^ (row mod 8): 16 lanes read from all banks (no conflicts
// counted). The loads for the steps to come are issued while reading and waited for
// with vmcnt(4), the youngest unit left in flight, two to three phases before use.
//
// Measured, 8192 x 32000 x 4096 with the loss's statistics behind it: 1.65 ms, 1,300
// TFLOP/s (the library's product of that shape with its bf16 result stored 1,360); a
// double buffer of both operands with one barrier a step 957; a ring of four stages of
// 32 values (rows of 64 bytes: twice the L2 requests) 1,260; four units released by
// halves of A's rows 1,286; the loads between the MFMAs 1,114, at their head 1,135.
// The clock falls to 1.65 GHz under this load; MFMAs are busy 64 to 70% of it.
//
// Turned operands come as lines of 512 bytes, 64 of them a unit, and leave LDS through
// ds_read_b64_tr_b16, twice as many reads of half the size. 8192 x 8192 x 4096: one
// operand turned 398 us (both along the axis 363), both turned 400 to 410 (371); copies
// that lie along the axis cost more than that (of dz while it is formed 25 us, of the
// classes 30, of the rows 23): a whole backward 4.85 ms against 4.9, and 5.6 against 5.85
// where classes are many; narrow ones gain 5 to 18%.
//
// Small tiles, 128 x 128 by four wavefronts of 64 x 64 and two workgroups a CU, for
// products of few large ones: the same ring at half the size, one barrier a step; the
// other workgroup's wavefront fills a SIMD's pauses.
#pragma once

#include "common.h"

namespace cign {
namespace ntgemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;   // values of a row in LDS at a time; rows are a multiple of it
constexpr int kUnits = 5;   // LDS: a ring of kStep values of a tile's rows of A or of B

// A workgroup's tile of TA rows of A by TB of B, WA x WB wavefronts.
template <int TA_, int TB_, int WA_, int WB_>
struct Shape {
  static constexpr int TA = TA_, TB = TB_, WA = WA_, WB = WB_;
  static constexpr int kThreads = WA * WB * kWave;
  static constexpr int FA = TA / WA / 16, FB = TB / WB / 16;  // 16 x 16 results of a wavefront
  static constexpr bool kPaired = WA * WB == 8;               // two wavefronts a SIMD, in turn
  static constexpr int kUnitBytes = TA * kStep * 2;
  static constexpr int kLdsBytes = kUnits * kUnitBytes;
  static constexpr int kGroups = kPaired ? 1 : 2;             // workgroups a CU
  static_assert(TA == TB && TA == WA * WB * 32, "a wavefront brings 32 rows of each operand");
};
using Large = Shape<256, 256, 2, 4>;
using Small = Shape<128, 128, 2, 2>;

// A matrix of bf16 values of `rows` rows along the summed axis, ld values apart,
// 16-byte aligned, of a multiple of kStep values (zeros beyond their own); `part` values
// on lies the next part of values held in several (split float32). Turned: as it stands
// the summed axis runs over its lines, of `width` values that may be read (a multiple of
// 8; value r of a line belongs to row r), and `depth` lines may be read: the last one is
// read again beyond them, where the other operand is zero.
struct Operand {
  const uint16_t* p;
  int64_t rows;
  int64_t ld;
  int64_t part;
  int64_t width = 0, depth = 0;
};

// Place of a wavefront's results: four consecutive rows of A by one row of B a lane.
template <class S>
struct Place {
  int64_t a0, b0;
  __device__ Place(int ia, int ib) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
    a0 = static_cast<int64_t>(ia) * S::TA + (w % S::WA) * (S::TA / S::WA) + (l >> 4) * 4;
    b0 = static_cast<int64_t>(ib) * S::TB + (w / S::WA) * (S::TB / S::WB) + (l & 15);
  }
  __device__ __forceinline__ int64_t a(int fa) const { return a0 + fa * 16; }
  __device__ __forceinline__ int64_t b(int fb) const { return b0 + fb * 16; }
};

// Tile of workgroup id: workgroups go round the 8 XCDs, each of which takes a
// contiguous run of tiles, in bands of 8 tiles of B, tile of A by tile of A: the 32
// tiles at work on an XCD share 4 tiles of A and 8 of B in its L2.
__device__ __forceinline__ void tile_of(int id, int ta, int tb, int& ia, int& ib) {
  const int total = ta * tb, x = id & 7, k = id >> 3;
  const int each = total >> 3, more = total & 7;
  const int t = x * each + min(x, more) + k;
  const int band = t / (8 * ta), rest = t - band * 8 * ta;
  const int wide = min(8, tb - band * 8);
  ia = rest / wide;
  ib = band * 8 + rest % wide;
}

typedef __attribute__((address_space(1))) const void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// Which parts of A and B a segment multiplies, the smallest products first. A step's
// segments follow each other, since they share parts that the caches still hold (125
// rows against 126,733 classes of 1184 float32, gradients: 1.91 ms segment by segment,
// 1.71 so).
__device__ __forceinline__ int seg_a(int s) { return (0x001102 >> (4 * s)) & 0xF; }
__device__ __forceinline__ int seg_b(int s) { return (0x010120 >> (4 * s)) & 0xF; }

// The fragments of half a step from LDS, waited for in the same statement.
__device__ __forceinline__ void read_both(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[8], bf16x8 (&b)[4]) {
  asm volatile(
      "ds_read_b128 %0, %13\n"
      "ds_read_b128 %1, %13 offset:2048\n"
      "ds_read_b128 %2, %13 offset:4096\n"
      "ds_read_b128 %3, %13 offset:6144\n"
      "ds_read_b128 %4, %12\n"
      "ds_read_b128 %5, %12 offset:2048\n"
      "ds_read_b128 %6, %12 offset:4096\n"
      "ds_read_b128 %7, %12 offset:6144\n"
      "ds_read_b128 %8, %12 offset:8192\n"
      "ds_read_b128 %9, %12 offset:10240\n"
      "ds_read_b128 %10, %12 offset:12288\n"
      "ds_read_b128 %11, %12 offset:14336\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]),
        "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7])
      : "v"(at_a), "v"(at_b)
      : "memory");
}
__device__ __forceinline__ void read_both(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[4], bf16x8 (&b)[4]) {
  asm volatile(
      "ds_read_b128 %0, %9\n"
      "ds_read_b128 %1, %9 offset:2048\n"
      "ds_read_b128 %2, %9 offset:4096\n"
      "ds_read_b128 %3, %9 offset:6144\n"
      "ds_read_b128 %4, %8\n"
      "ds_read_b128 %5, %8 offset:2048\n"
      "ds_read_b128 %6, %8 offset:4096\n"
      "ds_read_b128 %7, %8 offset:6144\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3])
      : "v"(at_a), "v"(at_b)
      : "memory");
}

// Fragments of turned units: sixteen lanes' 8 bytes of four lines come back as four
// lines of one value a lane, so two reads, four lines apart (OFF bytes), give a lane its
// eight. Fragment f lies at the first one's place ^ 32 f (the chunks' places are an xor).
// All of half a step's in one statement, waited for once: three waits took a tenth more
// of the whole product.
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <int N>
__device__ __forceinline__ void join(const s16x4 (&lo)[N], const s16x4 (&hi)[N], bf16x8 (&v)[N]) {
#pragma unroll
  for (int f = 0; f < N; ++f)
    v[f] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo[f], hi[f], 0, 1, 2, 3, 4, 5, 6, 7));
}
// A turned, B as it stands
template <int OFF>
__device__ __forceinline__ void read_turned_a(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[8], bf16x8 (&b)[4]) {
  s16x4 la[8], ha[8];
  asm volatile(
      "ds_read_b128 %0, %20\n"
      "ds_read_b128 %1, %20 offset:2048\n"
      "ds_read_b128 %2, %20 offset:4096\n"
      "ds_read_b128 %3, %20 offset:6144\n"
      "ds_read_b64_tr_b16 %4, %21\n"
      "ds_read_b64_tr_b16 %5, %21 offset:%29\n"
      "ds_read_b64_tr_b16 %6, %22\n"
      "ds_read_b64_tr_b16 %7, %22 offset:%29\n"
      "ds_read_b64_tr_b16 %8, %23\n"
      "ds_read_b64_tr_b16 %9, %23 offset:%29\n"
      "ds_read_b64_tr_b16 %10, %24\n"
      "ds_read_b64_tr_b16 %11, %24 offset:%29\n"
      "ds_read_b64_tr_b16 %12, %25\n"
      "ds_read_b64_tr_b16 %13, %25 offset:%29\n"
      "ds_read_b64_tr_b16 %14, %26\n"
      "ds_read_b64_tr_b16 %15, %26 offset:%29\n"
      "ds_read_b64_tr_b16 %16, %27\n"
      "ds_read_b64_tr_b16 %17, %27 offset:%29\n"
      "ds_read_b64_tr_b16 %18, %28\n"
      "ds_read_b64_tr_b16 %19, %28 offset:%29\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(la[0]), "=&v"(ha[0]),
        "=&v"(la[1]), "=&v"(ha[1]), "=&v"(la[2]), "=&v"(ha[2]), "=&v"(la[3]), "=&v"(ha[3]),
        "=&v"(la[4]), "=&v"(ha[4]), "=&v"(la[5]), "=&v"(ha[5]), "=&v"(la[6]), "=&v"(ha[6]),
        "=&v"(la[7]), "=&v"(ha[7])
      : "v"(at_b), "v"(at_a), "v"(at_a ^ 32), "v"(at_a ^ 64), "v"(at_a ^ 96), "v"(at_a ^ 128),
        "v"(at_a ^ 160), "v"(at_a ^ 192), "v"(at_a ^ 224), "n"(OFF)
      : "memory");
  join(la, ha, a);
}
template <int OFF>
__device__ __forceinline__ void read_turned_a(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[4], bf16x8 (&b)[4]) {
  s16x4 la[4], ha[4];
  asm volatile(
      "ds_read_b128 %0, %12\n"
      "ds_read_b128 %1, %12 offset:2048\n"
      "ds_read_b128 %2, %12 offset:4096\n"
      "ds_read_b128 %3, %12 offset:6144\n"
      "ds_read_b64_tr_b16 %4, %13\n"
      "ds_read_b64_tr_b16 %5, %13 offset:%17\n"
      "ds_read_b64_tr_b16 %6, %14\n"
      "ds_read_b64_tr_b16 %7, %14 offset:%17\n"
      "ds_read_b64_tr_b16 %8, %15\n"
      "ds_read_b64_tr_b16 %9, %15 offset:%17\n"
      "ds_read_b64_tr_b16 %10, %16\n"
      "ds_read_b64_tr_b16 %11, %16 offset:%17\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3]), "=&v"(la[0]), "=&v"(ha[0]),
        "=&v"(la[1]), "=&v"(ha[1]), "=&v"(la[2]), "=&v"(ha[2]), "=&v"(la[3]), "=&v"(ha[3])
      : "v"(at_b), "v"(at_a), "v"(at_a ^ 32), "v"(at_a ^ 64), "v"(at_a ^ 96), "n"(OFF)
      : "memory");
  join(la, ha, a);
}
// both turned
template <int OFF>
__device__ __forceinline__ void read_turned(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[8], bf16x8 (&b)[4]) {
  s16x4 la[8], ha[8], lb[4], hb[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %24\n"
      "ds_read_b64_tr_b16 %1, %24 offset:%36\n"
      "ds_read_b64_tr_b16 %2, %25\n"
      "ds_read_b64_tr_b16 %3, %25 offset:%36\n"
      "ds_read_b64_tr_b16 %4, %26\n"
      "ds_read_b64_tr_b16 %5, %26 offset:%36\n"
      "ds_read_b64_tr_b16 %6, %27\n"
      "ds_read_b64_tr_b16 %7, %27 offset:%36\n"
      "ds_read_b64_tr_b16 %8, %28\n"
      "ds_read_b64_tr_b16 %9, %28 offset:%36\n"
      "ds_read_b64_tr_b16 %10, %29\n"
      "ds_read_b64_tr_b16 %11, %29 offset:%36\n"
      "ds_read_b64_tr_b16 %12, %30\n"
      "ds_read_b64_tr_b16 %13, %30 offset:%36\n"
      "ds_read_b64_tr_b16 %14, %31\n"
      "ds_read_b64_tr_b16 %15, %31 offset:%36\n"
      "ds_read_b64_tr_b16 %16, %32\n"
      "ds_read_b64_tr_b16 %17, %32 offset:%36\n"
      "ds_read_b64_tr_b16 %18, %33\n"
      "ds_read_b64_tr_b16 %19, %33 offset:%36\n"
      "ds_read_b64_tr_b16 %20, %34\n"
      "ds_read_b64_tr_b16 %21, %34 offset:%36\n"
      "ds_read_b64_tr_b16 %22, %35\n"
      "ds_read_b64_tr_b16 %23, %35 offset:%36\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lb[0]), "=&v"(hb[0]), "=&v"(lb[1]), "=&v"(hb[1]), "=&v"(lb[2]), "=&v"(hb[2]),
        "=&v"(lb[3]), "=&v"(hb[3]), "=&v"(la[0]), "=&v"(ha[0]), "=&v"(la[1]), "=&v"(ha[1]),
        "=&v"(la[2]), "=&v"(ha[2]), "=&v"(la[3]), "=&v"(ha[3]), "=&v"(la[4]), "=&v"(ha[4]),
        "=&v"(la[5]), "=&v"(ha[5]), "=&v"(la[6]), "=&v"(ha[6]), "=&v"(la[7]), "=&v"(ha[7])
      : "v"(at_b), "v"(at_b ^ 32), "v"(at_b ^ 64), "v"(at_b ^ 96), "v"(at_a), "v"(at_a ^ 32),
        "v"(at_a ^ 64), "v"(at_a ^ 96), "v"(at_a ^ 128), "v"(at_a ^ 160), "v"(at_a ^ 192), "v"(at_a ^ 224),
        "n"(OFF)
      : "memory");
  join(lb, hb, b);
  join(la, ha, a);
}
template <int OFF>
__device__ __forceinline__ void read_turned(uint32_t at_a, uint32_t at_b, bf16x8 (&a)[4], bf16x8 (&b)[4]) {
  s16x4 la[4], ha[4], lb[4], hb[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n"
      "ds_read_b64_tr_b16 %1, %16 offset:%24\n"
      "ds_read_b64_tr_b16 %2, %17\n"
      "ds_read_b64_tr_b16 %3, %17 offset:%24\n"
      "ds_read_b64_tr_b16 %4, %18\n"
      "ds_read_b64_tr_b16 %5, %18 offset:%24\n"
      "ds_read_b64_tr_b16 %6, %19\n"
      "ds_read_b64_tr_b16 %7, %19 offset:%24\n"
      "ds_read_b64_tr_b16 %8, %20\n"
      "ds_read_b64_tr_b16 %9, %20 offset:%24\n"
      "ds_read_b64_tr_b16 %10, %21\n"
      "ds_read_b64_tr_b16 %11, %21 offset:%24\n"
      "ds_read_b64_tr_b16 %12, %22\n"
      "ds_read_b64_tr_b16 %13, %22 offset:%24\n"
      "ds_read_b64_tr_b16 %14, %23\n"
      "ds_read_b64_tr_b16 %15, %23 offset:%24\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lb[0]), "=&v"(hb[0]), "=&v"(lb[1]), "=&v"(hb[1]), "=&v"(lb[2]), "=&v"(hb[2]),
        "=&v"(lb[3]), "=&v"(hb[3]), "=&v"(la[0]), "=&v"(ha[0]), "=&v"(la[1]), "=&v"(ha[1]),
        "=&v"(la[2]), "=&v"(ha[2]), "=&v"(la[3]), "=&v"(ha[3])
      : "v"(at_b), "v"(at_b ^ 32), "v"(at_b ^ 64), "v"(at_b ^ 96), "v"(at_a), "v"(at_a ^ 32),
        "v"(at_a ^ 64), "v"(at_a ^ 96), "n"(OFF)
      : "memory");
  join(lb, hb, b);
  join(la, ha, a);
}

// Where line k of a turned unit has its 16-byte chunks: chunk c at place c ^ place(k),
// so that the 16 lines of a read lie on all banks.
__device__ __forceinline__ int place_of(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) << 1; }

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The tile (ia, ib) of the product over ksteps steps, SEGS segments each; ends
// with a barrier behind the last use of lds. Rows past an operand's last repeat it:
// their results are not to be used.
template <class S, int SEGS, bool TURN_A = false, bool TURN_B = false>
__device__ __forceinline__ void product(const Operand& A, const Operand& B, int ia, int ib, int ksteps, char* lds,
                                        f32x4 (&acc)[S::FA][S::FB]) {
  constexpr int kUnitBytes = S::kUnitBytes;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane_id();
  // What a lane brings of a unit, four times 16 bytes: of eight rows an instruction,
  // chunk c at place c ^ (row mod 8); turned, of the lines that 1 KB holds.
  constexpr int kPlaces = S::TA / 8, kLines = kWave / kPlaces;
  const int64_t a0 = static_cast<int64_t>(ia) * S::TA, b0 = static_cast<int64_t>(ib) * S::TB;
  uint32_t oa[4], ob[4];
  const auto offsets = [&](auto TURN, const Operand& X, int64_t first, uint32_t (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (decltype(TURN)::value) {
        const int k = (w * 4 + j) * kLines + l / kPlaces;
        o[j] = static_cast<uint32_t>(k) * static_cast<uint32_t>(X.ld) +
               static_cast<uint32_t>(min(first + ((l % kPlaces) ^ place_of(k)) * 8, X.width - 8));
      } else {
        const int last = static_cast<int>(min(static_cast<int64_t>(S::TA), X.rows - first)) - 1;
        o[j] = static_cast<uint32_t>(min(w * 32 + j * 8 + (l >> 3), last)) * static_cast<uint32_t>(X.ld) +
               ((l & 7) ^ (l >> 3)) * 8;
      }
    }
  };
  offsets(std::integral_constant<bool, TURN_A>(), A, a0, oa);
  offsets(std::integral_constant<bool, TURN_B>(), B, b0, ob);
  const uint16_t* pa = TURN_A ? A.p : A.p + a0 * A.ld;
  const uint16_t* pb = TURN_B ? B.p : B.p + b0 * B.ld;
  const int total = ksteps * SEGS;
  // the next unit of each operand: its step, the step in its segment, its segment
  int na = 0, ka = 0, ga = 0, nb = 0, kb = 0, gb = 0;
  int slot = 0;  // of the next unit
  const auto to_lds = [&](auto TURN, const Operand& X, const uint16_t* src, int k, const uint32_t (&o)[4]) {
    char* to = lds + slot * kUnitBytes + w * 4096;
    src += decltype(TURN)::value ? k * static_cast<int64_t>(kStep) * X.ld : static_cast<int64_t>(k) * kStep;
    const int last = decltype(TURN)::value ? static_cast<int>(X.depth - static_cast<int64_t>(k) * kStep) - 1 : kStep;
    const auto bring = [&](int j, uint32_t at) {
      __builtin_amdgcn_global_load_lds((GlobalPtr)(src + at), (LdsPtr)(to + j * 1024), 16, 0, 0);
    };
    if (decltype(TURN)::value && last < kStep - 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // lines beyond the last one: that one again
        const int line = (w * 4 + j) * kLines + l / kPlaces;
        bring(j, o[j] - static_cast<uint32_t>(max(line - last, 0)) * static_cast<uint32_t>(X.ld));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) bring(j, o[j]);
    }
  };
  const auto next = [&](int& k, int& g) {
    if (++g == SEGS) {
      g = 0;
      ++k;
    }
    slot = slot == kUnits - 1 ? 0 : slot + 1;
  };
  const auto load_a = [&]() {
    if (na >= total) return;
    to_lds(std::integral_constant<bool, TURN_A>(), A, pa + (SEGS > 1 ? seg_a(ga) * A.part : 0), ka, oa);
    next(ka, ga);
    ++na;
  };
  const auto load_b = [&]() {
    if (nb >= total) return;
    to_lds(std::integral_constant<bool, TURN_B>(), B, pb + (SEGS > 1 ? seg_b(gb) * B.part : 0), kb, ob);
    next(kb, gb);
    ++nb;
  };
#pragma unroll
  for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
    for (int fb = 0; fb < S::FB; ++fb) acc[fa][fb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (total == 0) return;
  load_a();
  load_b();
  load_a();
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsPtr)lds));
  constexpr int kLineBytes = S::TA * 2;
  // a lane's first bytes of half a step's fragments, of the wavefront's rows from `first`
  const auto begin = [&](bool turned, int first, int half) {
    if (turned) {
      const int k = half * 32 + (l >> 4) * 8 + ((l & 15) >> 2);
      return base + k * kLineBytes + (((first / 8 + ((l & 3) >> 1)) ^ place_of(k)) << 4) + (l & 1) * 8;
    }
    const int row = l & 15;
    return base + (first + row) * 128 + (((half * 4 + (l >> 4)) ^ (row & 7)) << 4);
  };
  const int first_a = (w % S::WA) * (S::TA / S::WA), first_b = (w / S::WA) * (S::TB / S::WB);
  const uint32_t at_a[2] = {begin(TURN_A, first_a, 0), begin(TURN_A, first_a, 1)};
  const uint32_t at_b[2] = {begin(TURN_B, first_b, 0), begin(TURN_B, first_b, 1)};
  const bool second = S::kPaired && w >= 4;
  if (total > 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  barrier();
  if (second) barrier();
  const auto steps = [&](auto on) {
    using ON = decltype(on);
    uint32_t ua = 0, ub = kUnitBytes;  // units of this step
    for (int t = 0; t < total; ++t) {
      const bool more = t + 2 < total;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 a[S::FA], b[S::FB];
        if (h == 0) load_b();
        else load_a();
        static_assert(TURN_A || !TURN_B, "a turned B beside a turned A only");
        if constexpr (ON::value) {
          if constexpr (!TURN_A) read_both(at_a[h] + ua, at_b[h] + ub, a, b);
          else if constexpr (TURN_B) read_turned<4 * kLineBytes>(at_a[h] + ua, at_b[h] + ub, a, b);
          else read_turned_a<4 * kLineBytes>(at_a[h] + ua, at_b[h] + ub, a, b);
        }
        if (h == 1 && second) {
          if (more) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
          else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (S::kPaired) {
          barrier();
          __builtin_amdgcn_s_setprio(1);
        }
        if constexpr (ON::value) {
#pragma unroll
          for (int fa = 0; fa < S::FA; ++fa)
#pragma unroll
            for (int fb = 0; fb < S::FB; ++fb)
              acc[fa][fb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[fa], b[fb], acc[fa][fb], 0, 0, 0);
        }
        if (S::kPaired) __builtin_amdgcn_s_setprio(0);
        if (h == 1 && !second) {
          if (more) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
          else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (S::kPaired || h == 1) barrier();
      }
      ua = ua >= 3 * kUnitBytes ? ua - 3 * kUnitBytes : ua + 2 * kUnitBytes;
      ub = ub >= 3 * kUnitBytes ? ub - 3 * kUnitBytes : ub + 2 * kUnitBytes;
    }
  };
  // A wavefront whose results lie behind the last row of A or B only brings its part of
  // the units and keeps the barriers: a tile of up to half its rows takes 0.75 of a full
  // one's time (777 rows against 50,001 classes of 1001 float32, forward: 605 -> 570 us).
  if (a0 + first_a < A.rows && b0 + first_b < B.rows) steps(std::true_type());
  else steps(std::false_type());
  if (S::kPaired && !second) barrier();
  __syncthreads();
}

}  // namespace ntgemm
}  // namespace cign

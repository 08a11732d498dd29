// C[n][m] = sum over k of A[m][k] * B[n][k] for bfloat16 operands, accumulated in float32 on v_mfma_f32_16x16x32_bf16, for the products of the
// class loss (dppm_classloss.hip).  Either operand may be contiguous in k, or in m (n): then it is given as [k][m].
//
// A float32 operand comes as three bfloat16 planes (hi + mid + lo hold its 24 significant bits); the same loop then walks six pairs of
// planes per step of k (all products down to 2^-16 of the largest), which makes a float32-grade product at a sixth of the bfloat16 rate --
// above the 157 TFLOP/s of the float32 matrix instructions.
//
// A workgroup holds a BM x BN tile; WGM x WGN waves hold WM x WN each.  Steps of 64 in k are brought to LDS by global_load_lds (16 bytes a
// lane, no registers) into a ring of stages, all but one of them ahead of the one that is multiplied.  A row of a stage is 128 bytes = one line
// = 8 chunks of 16; chunk c of row r lies in slot c ^ g, g = q ^ ((q >> 1 ^ q >> 2) & 1), q = (r >> 1) & 7: a 16-byte LDS read is served 16 lanes at
// a time, lanes 0-3, 12-15 and 20-27 together (then the others), that is rows 0-3 and 12-15 of one chunk with rows 4-11 of the next, and this
// way they fall on all banks (SQ_LDS_BANK_CONFLICT 0 in both kernels for float32, 2047 x 512 against 20011 classes; for bfloat16 1-9 % of the LDS cycles,
// all of it of tn_rows16; with g = r & 7 half of the LDS time was conflicts).  The DMA writes lanes side by side, so
// the swizzle is made on the global side: a lane fetches the chunk whose slot it fills.
//
// An operand that is contiguous in m lies in a stage as it comes, 64 rows of k with BM values, and its fragments are read by
// ds_read_b64_tr_b16: 16 lanes give the addresses of a block of 4 k by 16 m, 8 bytes each, and lane i gets column i's four values.  Two of them
// make the eight k of a lane.  32 lanes read 8 rows (k = 0-3 and 8-11, or 4 more) at once, 32 bytes each: the 32-byte blocks of a row are turned
// by (k & 3) + 4 (k >> 3 & 1), which puts them on all banks.
#pragma once
#include "dppm_common.h"

namespace dppm {

typedef __bf16 tn_frag __attribute__((ext_vector_type(8)));
typedef float tn_acc __attribute__((ext_vector_type(4)));

struct TnArgs {
  const uint16_t* A; const uint16_t* B;
  long lda, ldb;          // elements between rows (of m or n, or of k); multiples of 8, as the planes' distance
  long plane_a, plane_b;  // elements between planes
  int M, N, K, ksteps;       // ksteps = k / 64: operands contiguous in k are padded with zeros to whole steps
  int pairs;              // 1; 6 for float32 operands in three planes; 2 for one plane of A with two of B
  int splits;             // parts that the steps of k are dealt to
  int tiles_m, tiles_n;
};

// plane of A and of B in each of the six products, four bits each, largest product first: (0,0) (0,1) (1,0) (0,2) (2,0) (1,1)
constexpr uint32_t kPairA = 0x120100u, kPairB = 0x102010u;

template <int BM_, int BN_, int WGM_, int WGN_, int STAGES_>
struct TnTile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, WAVES = WGM * WGN, NT = WAVES * 64;
  static constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NI = WN / 16;
  static constexpr int STAGES = STAGES_, STAGE = (BM + BN) * 128;
  static constexpr int OUT_PITCH = WM * 4 + 16;                    // a row of the epilogue's image: WM float32 values and a gap
  static constexpr int OUT = WAVES * 32 * OUT_PITCH;
  static constexpr int LDS = STAGES * STAGE > OUT ? STAGES * STAGE : OUT;
  static_assert((BM * 8) % NT == 0 && (BN * 8) % NT == 0 && NT % 128 == 0 && STAGES >= 2 && LDS <= 160 * 1024, "whole rounds of loads");
};

// Which tile a workgroup takes.  Workgroups go round the 8 dies; tiles that follow each other on one die share operand rows in its L2:
// the die's stretch of the tile list is contiguous, and the list runs down columns of GROUP tiles.  (The largest class loss, all of it:
// 21.2 ms with 4, 21.4 with 8, 23.9 with 16.)
__device__ __forceinline__ void tn_tile_of(int id, int count, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = count / 8, rest = count % 8, die = id % 8, at = id / 8;
  const int t = die * per + (die < rest ? die : rest) + at;        // dies 0 .. rest-1 hold one tile more
  constexpr int GROUP = 4;
  const int band = t / (GROUP * tiles_n), first = band * GROUP;
  const int rows = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int in = t - band * GROUP * tiles_n;
  tm = first + in % rows;
  tn = in / rows;
}

template <int N> struct Int { static constexpr int value = N; };

// what chunk numbers of a row are turned by
__device__ __forceinline__ int tn_turn(int row) {
  const int q = (row >> 1) & 7;
  return q ^ (((q >> 1) ^ (q >> 2)) & 1);
}

// Offsets in bytes of the 16-byte chunks a thread brings in, one a round, from an operand whose tile begins at row (or column) `first` of `count`.
// Contiguous in k: WIDTH rows of 8 chunks; rows behind the last repeat it, their results are not kept.  Else: 64 rows of k with WIDTH / 8
// chunks; chunks behind the pitch repeat its last, and in the last step rows of k behind `ks` repeat the last, where the other operand
// holds zeros.
template <int WIDTH, int NT, bool TR>
__device__ __forceinline__ void tn_offsets(uint32_t (&off)[WIDTH * 8 / NT], long ld, int first, int count, int ks) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int r = 0; r < WIDTH * 8 / NT; ++r) {
    if constexpr (TR) {
      constexpr int PER = WIDTH / 8;
      const int k = (r * NT + tid) / PER, turn = ((k & 3) | ((k >> 1) & 4)) << 1;
      const int c = ((tid % PER) ^ turn), last = (int)(ld / 8) - 1 - first / 8;
      off[r] = (uint32_t)(((long)(k < ks ? k : ks - 1) * ld + (c < last ? c : last) * 8) * 2);
    } else {
      const int row = tid >> 3, chunk = (tid & 7) ^ tn_turn(row), x = row + r * (NT / 8), last = count - 1 - first;
      off[r] = (uint32_t)(((long)(x < last ? x : last) * ld + chunk * 8) * 2);
    }
  }
}

// TRA, TRB: the operand is contiguous in m (n)
template <class T, bool TRA, bool TRB>
__device__ __forceinline__ void tn_product(const TnArgs& g, char* lds, int m0, int n0, int it0, int it1, tn_acc (&acc)[T::MI][T::NI]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % T::WGM, wn = wave / T::WGM;
  constexpr int RA = T::BM * 8 / T::NT, RB = T::BN * 8 / T::NT;   // rounds of loads
  uint32_t off_a[RA], off_b[RB];
  tn_offsets<T::BM, T::NT, TRA>(off_a, g.lda, m0, g.M, 64);
  tn_offsets<T::BN, T::NT, TRB>(off_b, g.ldb, n0, g.N, 64);
  int pair = it0 % g.pairs;
  long step = it0 / g.pairs;
  const uint16_t *base_a = g.A + (TRA ? (long)m0 : (long)m0 * g.lda), *base_b = g.B + (TRB ? (long)n0 : (long)n0 * g.ldb);
  const char *src_a, *src_b;
  const auto seek = [&] {      // where the next stage comes from
    src_a = reinterpret_cast<const char*>(base_a + (long)((kPairA >> (4 * pair)) & 15u) * g.plane_a + (TRA ? step * 64 * g.lda : step * 64));
    src_b = reinterpret_cast<const char*>(base_b + (long)((kPairB >> (4 * pair)) & 15u) * g.plane_b + (TRB ? step * 64 * g.ldb : step * 64));
    if (step == g.ksteps - 1) {      // (and that is where these offsets stay)
      const int left = g.K - (int)step * 64;
      if (TRA && left < 64) tn_offsets<T::BM, T::NT, TRA>(off_a, g.lda, m0, g.M, left);
      if (TRB && left < 64) tn_offsets<T::BN, T::NT, TRB>(off_b, g.ldb, n0, g.N, left);
    }
    if (++pair == g.pairs) { pair = 0; ++step; }
  };
  const auto load = [&](int stage, int r0, int r1) {    // rounds r0 .. r1 - 1 of A's followed by B's
    char* to = lds + stage * T::STAGE + wave * 1024;
#pragma unroll
    for (int r = 0; r < RA + RB; ++r)
      if (r >= r0 && r < r1)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(r < RA ? src_a + off_a[r < RA ? r : 0] : src_b + off_b[r < RA ? 0 : r - RA]),
                                         (__attribute__((address_space(3))) void*)(to + r * T::NT * 16), 16, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.f;
  if (it0 >= it1) return;
  // Contiguous in k: this lane's row is lane & 15 of 16, its chunk 4 ks + (lane >> 4) for the two halves ks of a stage.
  uint32_t slot[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) slot[ks] = (uint32_t)((lane & 15) * 128 + (((4 * ks + (lane >> 4)) ^ tn_turn(lane & 15)) * 16));
  // Else: the address this lane gives for row 8 (lane >> 4) + (lane >> 2 & 3) of k, in the block of 16 m that its turn makes of block i
  const uint32_t block = ((lane >> 2) & 3) | ((lane >> 2) & 4), row = (uint32_t)(8 * (lane >> 4) + ((lane >> 2) & 3)), within = (lane & 3) * 8;
  uint32_t tr_a[TRA ? T::MI : 1], tr_b[TRB ? T::NI : 1];
#pragma unroll
  for (int i = 0; i < (TRA ? T::MI : 1); ++i) tr_a[i] = row * (T::BM * 2) + (((wm * T::MI + i) ^ block) * 32) + within;
#pragma unroll
  for (int j = 0; j < (TRB ? T::NI : 1); ++j) tr_b[j] = T::BM * 128 + row * (T::BN * 2) + (((wn * T::NI + j) ^ block) * 32) + within;
  const uint32_t frag_a = wm * T::WM * 128, frag_b = T::BM * 128 + wn * T::WN * 128;
  constexpr int HALF = T::MI / 2;
  static_assert(!TRA || HALF == 4 || HALF == 2, "");
  static_assert(!TRB || T::NI % 4 == 0, "");
  tn_frag a[T::MI], b[2][T::NI];
  // The builtin for these reads makes the compiler wait for every global_load_lds in flight first, so they are written out, with their wait:
  // nothing is in flight when the block ends.  The other wave of the SIMD multiplies meanwhile.
  typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
  const auto turned4 = [&](tn_frag* out, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, auto pitch) {
    u32x2v r0, r1, r2, r3, r4, r5, r6, r7;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3), "=&v"(r4), "=&v"(r5), "=&v"(r6), "=&v"(r7)
        : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(4 * decltype(pitch)::value));
    out[0] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r0, r1, 0, 1, 2, 3));
    out[1] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r2, r3, 0, 1, 2, 3));
    out[2] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r4, r5, 0, 1, 2, 3));
    out[3] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r6, r7, 0, 1, 2, 3));
  };
  const auto turned2 = [&](tn_frag* out, uint32_t a0, uint32_t a1, auto pitch) {
    u32x2v r0, r1, r2, r3;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
        "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
        : "v"(a0), "v"(a1), "n"(4 * decltype(pitch)::value));
    out[0] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r0, r1, 0, 1, 2, 3));
    out[1] = __builtin_bit_cast(tn_frag, __builtin_shufflevector(r2, r3, 0, 1, 2, 3));
  };
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const auto read_a = [&](int i0, int i1, int stage, int ks) {
    if constexpr (TRA) {
      const uint32_t s = lds_at + stage * T::STAGE + ks * 32 * (T::BM * 2);
#pragma unroll
      for (int i = 0; i < T::MI; i += HALF)      // a half is 4 or 2 fragments
        if (i == i0) {
          if constexpr (HALF == 4) turned4(a + i, s + tr_a[i], s + tr_a[i + 1], s + tr_a[i + 2], s + tr_a[i + 3], Int<T::BM * 2>{});
          else turned2(a + i, s + tr_a[i], s + tr_a[i + 1], Int<T::BM * 2>{});
        }
    } else {
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
        if (i >= i0 && i < i1) a[i] = *reinterpret_cast<const tn_frag*>(lds + stage * T::STAGE + frag_a + slot[ks] + i * 2048);
    }
  };
  const auto read_b = [&](int stage, int ks) {
    if constexpr (TRB) {
      const uint32_t s = lds_at + stage * T::STAGE + ks * 32 * (T::BN * 2);
#pragma unroll
      for (int j = 0; j < T::NI; j += 4) turned4(b[ks] + j, s + tr_b[j], s + tr_b[j + 1], s + tr_b[j + 2], s + tr_b[j + 3], Int<T::BN * 2>{});
    } else {
#pragma unroll
      for (int j = 0; j < T::NI; ++j) b[ks][j] = *reinterpret_cast<const tn_frag*>(lds + stage * T::STAGE + frag_b + slot[ks] + j * 2048);
    }
  };
  const auto multiply = [&](int i0, int i1, int ks) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < T::MI; ++i)
      if (i >= i0 && i < i1) {
#pragma unroll
        for (int j = 0; j < T::NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[ks][j], acc[i][j], 0, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Loads complete in order: with the loads of AHEAD stages behind it outstanding, a stage has landed.
  constexpr int R = RA + RB, AHEAD = T::STAGES - 2, OUTSTANDING = AHEAD * R;
  static_assert(OUTSTANDING < 64, "vmcnt");
  const int count = it1 - it0;
#pragma unroll
  for (int p = 0; p < T::STAGES - 1; ++p)
    if (p < count) { seek(); load(p, 0, R); }
  if (count >= T::STAGES - 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(OUTSTANDING) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  read_a(0, HALF, 0, 0);
  read_b(0, 0);
  int stage = 0, spare = T::STAGES - 1;     // the stage that is multiplied, the one that is filled
  for (int it = 0; it < count; ++it) {
    // Four quarters of a stage: half of the rows of m times half of k; the next quarter's fragments are read while one is multiplied.  Half of
    // the next stage's loads go out in the first quarter, half in the second (all in the first: 4 % longer; over three: 5 %).
    const bool more = it + T::STAGES - 1 < count;
    if (more) { seek(); load(spare, 0, R / 2); }
    read_a(HALF, T::MI, stage, 0);
    multiply(0, HALF, 0);
    if (more) load(spare, R / 2, R);
    read_a(0, HALF, stage, 1);
    read_b(stage, 1);
    multiply(HALF, T::MI, 0);
    read_a(HALF, T::MI, stage, 1);
    multiply(0, HALF, 1);
    spare = stage;
    stage = stage + 1 == T::STAGES ? 0 : stage + 1;
    // The next stage has landed, and nobody reads this one any more.  (Behind the last stage another is read once for nothing.)
    if (more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(OUTSTANDING) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    read_a(0, HALF, stage, 0);
    read_b(stage, 0);
    multiply(HALF, T::MI, 1);
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");     // the reads for nothing, before the stages are used for something else
}

// 32 n of a wave's result through LDS, so that memory sees whole rows of m.  A lane holds n = 16 j + (lane & 15) and m = 16 i + 4 (lane >> 4)
// + 0..3.  `emit(row, m, eight values)` is called for 32 rows n from 32 `block` on, with m in steps of 8 side by side over the lanes.
template <class T, class Emit>
__device__ __forceinline__ void tn_rows(char* lds, const tn_acc (&acc)[T::MI][T::NI], int block, Emit emit) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* img = lds + wave * 32 * T::OUT_PITCH;
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
      if (j / 2 == block) *reinterpret_cast<tn_acc*>(img + ((j & 1) * 16 + (lane & 15)) * T::OUT_PITCH + (16 * i + 4 * (lane >> 4)) * 4) = acc[i][j];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  constexpr int PER_ROW = T::WM / 8, ROWS = 64 / PER_ROW;
#pragma unroll
  for (int r = 0; r < 32; r += ROWS) {
    const int row = r + lane / PER_ROW, m = (lane % PER_ROW) * 8;
    const tn_acc* p = reinterpret_cast<const tn_acc*>(img + row * T::OUT_PITCH + m * 4);
    const tn_acc x = p[0], y = p[1];
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    emit(row, m, v);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// The same with the values packed to 16 bits on the way in, which halves the LDS traffic
// (4099 x 1000 bfloat16, 50001 classes: 1.525 -> 1.510 ms): pack(lo, hi) makes a word of two,
// emit(row, m, word[4]) gets eight values.
template <class T, class Pack, class Emit>
__device__ __forceinline__ void tn_rows16(char* lds, const tn_acc (&acc)[T::MI][T::NI], int block, Pack pack, Emit emit) {
  typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
  constexpr int PITCH = T::WM * 2 + 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* img = lds + wave * 32 * PITCH;
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
      if (j / 2 == block)
        *reinterpret_cast<u32x2v*>(img + ((j & 1) * 16 + (lane & 15)) * PITCH + (16 * i + 4 * (lane >> 4)) * 2) =
            u32x2v{pack(acc[i][j][0], acc[i][j][1]), pack(acc[i][j][2], acc[i][j][3])};
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  constexpr int PER_ROW = T::WM / 8, ROWS = 64 / PER_ROW;
#pragma unroll
  for (int r = 0; r < 32; r += ROWS) {
    const int row = r + lane / PER_ROW, m = (lane % PER_ROW) * 8;
    emit(row, m, *reinterpret_cast<const u32x4v*>(img + row * PITCH + m * 2));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

}  // namespace dppm

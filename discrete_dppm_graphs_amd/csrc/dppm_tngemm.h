// C[n][m] = sum over k of A[m][k] * B[n][k] for bfloat16 operands that are both contiguous in k, accumulated in float32 on
// v_mfma_f32_32x32x16_bf16, for the products of the class loss (dppm_classloss.hip).
//
// A float32 operand comes as three bfloat16 planes (hi + mid + lo hold its 24 significant bits); the same loop then walks six pairs of
// planes per step of k (all products down to 2^-16 of the largest), which makes a float32-grade product at a sixth of the bfloat16 rate --
// above the 157 TFLOP/s of the float32 matrix instructions.
//
// A workgroup holds a BM x BN tile; WGM x WGN waves hold WM x WN each.  Steps of 64 in k are brought to LDS by global_load_lds (16 bytes a
// lane, no registers), into the other of two stages while one is multiplied.  A row of a stage is 128 bytes = 8 chunks of 16; chunk c of row
// r lies in slot c ^ (r & 7), so that the 16-byte fragment reads of 8 rows at a time fall on all banks.  The DMA writes lanes side by side, so
// the swizzle is made on the global side: a lane fetches the chunk whose slot it fills.
#pragma once
#include "dppm_common.h"

namespace dppm {

typedef __bf16 tn_frag __attribute__((ext_vector_type(8)));
typedef float tn_acc __attribute__((ext_vector_type(16)));

struct TnArgs {
  const uint16_t* A; const uint16_t* B;
  long lda, ldb;          // elements between rows; multiples of 8, as the planes' distance
  long plane_a, plane_b;  // elements between planes
  int M, N, ksteps;       // ksteps = k / 64: operands are padded with zeros to whole steps
  int pairs;              // 1, or 6 for float32 operands in three planes
  int splits;             // parts that the steps of k are dealt to
  int tiles_m, tiles_n;
};

// plane of A and of B in each of the six products, four bits each, largest product first: (0,0) (0,1) (1,0) (0,2) (2,0) (1,1)
constexpr uint32_t kPairA = 0x120100u, kPairB = 0x102010u;

template <int BM_, int BN_, int WGM_, int WGN_>
struct TnTile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, WAVES = WGM * WGN, NT = WAVES * 64;
  static constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NI = WN / 32;
  static constexpr int STAGE = (BM + BN) * 128;
  static constexpr int OUT_PITCH = WM * 4 + 16;                    // a row of the epilogue's image: WM float32 values and a gap
  static constexpr int OUT = WAVES * 32 * OUT_PITCH;
  static constexpr int LDS = 2 * STAGE > OUT ? 2 * STAGE : OUT;
  static_assert((BM * 8) % NT == 0 && (BN * 8) % NT == 0, "whole rounds of loads");
};

// Which tile a workgroup takes.  Workgroups go round the 8 dies; tiles that follow each other on one die share operand rows in its L2:
// the die's stretch of the tile list is contiguous, and the list runs down columns of GROUP tiles.
__device__ __forceinline__ void tn_tile_of(int id, int count, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = count / 8, rest = count % 8, die = id % 8, at = id / 8;
  const int t = die * per + (die < rest ? die : rest) + at;        // dies 0 .. rest-1 hold one tile more
  constexpr int GROUP = 8;
  const int band = t / (GROUP * tiles_n), first = band * GROUP;
  const int rows = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  const int in = t - band * GROUP * tiles_n;
  tm = first + in % rows;
  tn = in / rows;
}

template <class T>
__device__ __forceinline__ void tn_product(const TnArgs& g, char* lds, int m0, int n0, int it0, int it1, tn_acc (&acc)[T::MI][T::NI]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % T::WGM, wn = wave / T::WGM;
  constexpr int RA = T::BM * 8 / T::NT, RB = T::BN * 8 / T::NT, ROWS = T::NT / 8;   // rounds of loads, rows of a round
  uint32_t off_a[RA], off_b[RB];
  {
    const int row = tid >> 3, chunk = (tid & 7) ^ (row & 7);
#pragma unroll
    for (int r = 0; r < RA; ++r) {
      const int x = row + r * ROWS, last = g.M - 1 - m0;
      off_a[r] = (uint32_t)(((long)(x < last ? x : last) * g.lda + chunk * 8) * 2);      // rows behind the last repeat it: their results are not kept
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int x = row + r * ROWS, last = g.N - 1 - n0;
      off_b[r] = (uint32_t)(((long)(x < last ? x : last) * g.ldb + chunk * 8) * 2);
    }
  }
  int pair = it0 % g.pairs;
  long step = it0 / g.pairs;
  const uint16_t *base_a = g.A + (long)m0 * g.lda, *base_b = g.B + (long)n0 * g.ldb;
  const auto load = [&](int stage) {
    const char* a = reinterpret_cast<const char*>(base_a + (long)((kPairA >> (4 * pair)) & 15u) * g.plane_a + step * 64);
    const char* b = reinterpret_cast<const char*>(base_b + (long)((kPairB >> (4 * pair)) & 15u) * g.plane_b + step * 64);
    char* to = lds + stage * T::STAGE + wave * 1024;
#pragma unroll
    for (int r = 0; r < RA; ++r)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a + off_a[r]),
                                       (__attribute__((address_space(3))) void*)(to + r * T::NT * 16), 16, 0, 0);
#pragma unroll
    for (int r = 0; r < RB; ++r)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(b + off_b[r]),
                                       (__attribute__((address_space(3))) void*)(to + T::BM * 128 + r * T::NT * 16), 16, 0, 0);
    if (++pair == g.pairs) { pair = 0; ++step; }
  };
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;
  if (it0 >= it1) return;
  uint32_t slot[4];     // byte of chunk 2 ks + (lane >> 5) in this lane's row, for the four k steps of a stage
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) slot[ks] = (uint32_t)(((lane & 31) * 128) + (((2 * ks + (lane >> 5)) ^ (lane & 7)) * 16));
  const uint32_t frag_a = wm * T::WM * 128, frag_b = T::BM * 128 + wn * T::WN * 128;
  load(0);
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  for (int it = it0; it < it1; ++it) {
    const int stage = (it - it0) & 1;
    if (it + 1 < it1) load(stage ^ 1);
    const char* s = lds + stage * T::STAGE;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      tn_frag a[T::MI], b[T::NI];
#pragma unroll
      for (int i = 0; i < T::MI; ++i) a[i] = *reinterpret_cast<const tn_frag*>(s + frag_a + i * 4096 + slot[ks]);
#pragma unroll
      for (int j = 0; j < T::NI; ++j) b[j] = *reinterpret_cast<const tn_frag*>(s + frag_b + j * 4096 + slot[ks]);
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int j = 0; j < T::NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
    }
    // the next stage has landed, and nobody reads this one any more
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
}

// One column block of 32 n of a wave's result through LDS, so that memory sees whole rows of m.  A lane holds n = lane & 31 and
// m = 32 i + 8 q + 4 (lane >> 5) + 0..3 for q = 0..3.  `emit(row n, m, eight values)` is called with m in steps of 8 side by side over the lanes.
template <class T, class Emit>
__device__ __forceinline__ void tn_rows(char* lds, const tn_acc (&acc)[T::MI][T::NI], int j, Emit emit) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* img = lds + wave * 32 * T::OUT_PITCH;
  typedef float f32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(img + (lane & 31) * T::OUT_PITCH + (32 * i + 8 * q + 4 * (lane >> 5)) * 4) =
          f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  constexpr int PER_ROW = T::WM / 8, ROWS = 64 / PER_ROW;
#pragma unroll
  for (int r = 0; r < 32; r += ROWS) {
    const int row = r + lane / PER_ROW, m = (lane % PER_ROW) * 8;
    const f32x4* p = reinterpret_cast<const f32x4*>(img + row * T::OUT_PITCH + m * 4);
    const f32x4 x = p[0], y = p[1];
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    emit(row, m, v);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

}  // namespace dppm

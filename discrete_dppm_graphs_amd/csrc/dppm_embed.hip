// A table of classes: out[t] = scale * W[id_t], and its gradient dW[v] = scale * sum over t with id_t = v of dout[t].
// An id outside [0, V) stands for no class (a padded position): its row of `out` is zero and it adds nothing to any gradient.
//
// Both are HBM-bound.  The lookup reads and writes each row once, 16 bytes a lane.  The gradient sorts the positions by class (a stable
// radix sort of (class, position) pairs), so that the rows of one class lie together and are summed in the order of their positions in
// float32 registers: no atomics, the same bits from call to call, and one write per row of dW.  A class with many positions is split over
// fixed chunks of the sorted order, whose partial rows a second launch joins, again in order.  Small tables and few positions need no sorting
// (embed_small_kernel, embed_range_kernel).
#include "dppm_common.h"

namespace dppm {
namespace {

template <class T> using glb = __attribute__((address_space(1))) T*;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // round to nearest even (v_cvt_pk_bf16_f32)
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// VEC values from / to memory, as float32.  VEC > 1: 16 bytes of the input's type, aligned.
template <bool BF, int VEC>
__device__ __forceinline__ void load_vec(const void* src, long at, float (&v)[VEC]) {
  if constexpr (BF && VEC == 8) {
    const u32x4 w = *(glb<const u32x4>)((glb<const uint16_t>)src + at);
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[2 * k] = bf16_lo(w[k]); v[2 * k + 1] = bf16_hi(w[k]); }
  } else if constexpr (BF) {
    static_assert(VEC == 1, "");
    v[0] = bf16_lo(((glb<const uint16_t>)src)[at]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      if constexpr (VEC >= 4) {
        const f32x4 w = *(glb<const f32x4>)((glb<const float>)src + at + k);
        v[k] = w.x; v[k + 1] = w.y; v[k + 2] = w.z; v[k + 3] = w.w;
      } else v[0] = ((glb<const float>)src)[at];
    }
  }
}
template <bool BF, int VEC>
__device__ __forceinline__ void store_vec(void* dst, long at, const float (&v)[VEC]) {
  if constexpr (BF) {
    const glb<uint16_t> q = (glb<uint16_t>)dst + at;
    if constexpr (VEC == 8) *(glb<u32x4>)q = u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    else if constexpr (VEC == 4) *(glb<u32x2>)q = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    else *q = to_bf16(v[0]);
  } else {
    const glb<float> q = (glb<float>)dst + at;
    if constexpr (VEC == 1) *q = v[0];
    else {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) *(glb<f32x4>)(q + k) = f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]};
    }
  }
}

// ------------------------------------------------------------------------------------------------ lookup
// `tpr` threads (a power of two, at most 256) walk a row; a workgroup holds 256 / tpr rows at a time and four such groups, whose loads
// are issued together.
constexpr int FWD_ROWS = 4;
template <bool BF, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* __restrict__ w, const int64_t* __restrict__ ids, float scale, void* __restrict__ out,
                                                        long T, long V, int D, int tpr_log2) {
  const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2, lane = threadIdx.x & (tpr - 1);
  const long t0 = (long)blockIdx.x * rpb * FWD_ROWS + (threadIdx.x >> tpr_log2);
  long id[FWD_ROWS];
#pragma unroll
  for (int r = 0; r < FWD_ROWS; ++r) {
    const long t = t0 + r * rpb;
    const long i = t < T ? ids[t] : -1;
    id[r] = i < V ? i : -1;
  }
  for (int c = lane * VEC; c < D; c += tpr * VEC) {
    float v[FWD_ROWS][VEC];
#pragma unroll
    for (int r = 0; r < FWD_ROWS; ++r) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[r][k] = 0.f;
      if (id[r] >= 0) load_vec<BF, VEC>(w, id[r] * D + c, v[r]);
    }
#pragma unroll
    for (int r = 0; r < FWD_ROWS; ++r) {
      const long t = t0 + r * rpb;
      if (t < T) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[r][k] *= scale;
        if (id[r] < 0) {   // 0 * scale would be NaN for an infinite scale
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[r][k] = 0.f;
        }
        store_vec<BF, VEC>(out, t * D + c, v[r]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ sorting positions by class
// Least significant digit first: count the digits of every tile, then place every pair at
//   (pairs with a smaller digit) + (pairs with the digit in earlier tiles) + (rank among the tile's pairs with the digit),
// which keeps the order of equal digits.  Classes without a row sort behind all others as class V.  The bits of V are shared evenly over
// as few passes as the digit's width allows.  Up to ONE_TILE positions one workgroup sorts alone in one launch, 10 bits a pass; more are
// cut into tiles of 1024 positions and up, 9 bits a pass and two launches each.
constexpr int ONE_BITS = 10, TILE_BITS = 9;
constexpr int MAX_TILES = 128;                 // every tile's placement reads the counts of all
constexpr int ONE_TILE = 8192;                 // 1024 threads x 8
constexpr int TILE = 1024;                     // 256 threads x 4

struct SortBufs { uint32_t *key[2], *pos[2]; };

__device__ __forceinline__ uint32_t class_key(const int64_t* ids, long t, long V) {
  const long i = ids[t];
  return (uint32_t)((i >= 0 && i < V) ? i : V);
}

template <int NT, int BITS>
struct RankShared { uint32_t cnt[NT / 64][1 << BITS]; uint32_t base[1 << BITS]; uint32_t wave[NT / 64]; };

// s.base: counts -> their exclusive prefix sum.  Called by every thread, between barriers of its own.
template <int NT, int BITS>
__device__ __forceinline__ void scan_digits(RankShared<NT, BITS>& s) {
  constexpr int E = ((1 << BITS) + NT - 1) / NT;     // digits of a thread
  static_assert(E * NT == (1 << BITS), "");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  uint32_t own[E], sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) { own[e] = s.base[threadIdx.x * E + e]; sum += own[e]; }
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  if (lane == 63) s.wave[wave] = incl;
  __syncthreads();
  uint32_t at = incl - sum;
  for (int w = 0; w < wave; ++w) at += s.wave[w];
#pragma unroll
  for (int e = 0; e < E; ++e) { s.base[threadIdx.x * E + e] = at; at += own[e]; }
  __syncthreads();
}

// Places NT * PER consecutive pairs from `begin` on (those before `n`).  s.base[d]: where the next pair with digit d goes, moved on for the
// next call; ALONE: these are all pairs, and s.base comes from their counts.  A wave takes 64 * PER consecutive pairs, 64 at a time; lanes
// with the same digit are found with one ballot per bit.
template <int NT, int BITS, int PER, bool FIRST, bool ALONE>
__device__ __forceinline__ void place(RankShared<NT, BITS>& s, const int64_t* ids, long V, const uint32_t* key_in, const uint32_t* pos_in, uint32_t* key_out,
                                      uint32_t* pos_out, long begin, long n, int shift, int bits) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t low = (1u << bits) - 1u;
  for (int i = threadIdx.x; i < (NT / 64) << BITS; i += NT) (&s.cnt[0][0])[i] = 0;
  uint32_t key[PER], pos[PER], rank[PER];
  const long at0 = begin + (long)wave * 64 * PER + lane;
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const long at = at0 + r * 64;
    key[r] = 0; pos[r] = 0;
    if (at < n) {
      if (FIRST) { key[r] = class_key(ids, at, V); pos[r] = (uint32_t)at; }
      else { key[r] = key_in[at]; pos[r] = pos_in[at]; }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    rank[r] = 0;
    if (at0 - lane + r * 64 >= n) continue;      // the whole wave is behind the end
    const bool in = at0 + r * 64 < n;
    const uint32_t d = (key[r] >> shift) & low;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t one = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? one : ~one;
    }
    const uint64_t before = same & ((1ull << lane) - 1ull);
    uint32_t seen = 0;
    if (in) seen = s.cnt[wave][d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    rank[r] = seen + __popcll(before);
    if (in && before == 0) s.cnt[wave][d] = seen + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  if (ALONE) {
    for (int d = threadIdx.x; d < (1 << BITS); d += NT) {
      uint32_t c = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) c += s.cnt[w][d];
      s.base[d] = c;
    }
    scan_digits(s);
  }
  for (int d = threadIdx.x; d < (1 << BITS); d += NT) {   // where each wave's pairs with the digit begin
    uint32_t b = s.base[d];
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      const uint32_t c = s.cnt[w][d];
      s.cnt[w][d] = b;
      b += c;
    }
    s.base[d] = b;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PER; ++r)
    if (at0 + r * 64 < n) {
      const uint32_t to = s.cnt[wave][(key[r] >> shift) & low] + rank[r];
      key_out[to] = key[r];
      pos_out[to] = pos[r];
    }
  __syncthreads();
}

__global__ __launch_bounds__(1024) void sort_one_kernel(const int64_t* __restrict__ ids, long T, long V, int passes, int bits, SortBufs b) {
  __shared__ RankShared<1024, ONE_BITS> s;
  place<1024, ONE_BITS, ONE_TILE / 1024, true, true>(s, ids, V, nullptr, nullptr, b.key[0], b.pos[0], 0, T, 0, bits);
  for (int p = 1; p < passes; ++p) {
    const int out = p & 1;
    place<1024, ONE_BITS, ONE_TILE / 1024, false, true>(s, ids, V, b.key[out ^ 1], b.pos[out ^ 1], b.key[out], b.pos[out], 0, T, bits * p, bits);
  }
}

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ key, long T, long V, int shift, int bits,
                                                         long tile, uint32_t* __restrict__ hist) {
  __shared__ uint32_t h[1 << TILE_BITS];
  for (int d = threadIdx.x; d < (1 << TILE_BITS); d += 256) h[d] = 0;
  __syncthreads();
  const uint32_t low = (1u << bits) - 1u;
  const long begin = blockIdx.x * tile, end = begin + tile < T ? begin + tile : T;
  for (long t = begin + threadIdx.x; t < end; t += 256) atomicAdd(&h[((FIRST ? class_key(ids, t, V) : key[t]) >> shift) & low], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < (1 << TILE_BITS); d += 256) hist[((long)blockIdx.x << TILE_BITS) + d] = h[d];
}

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_place_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ key_in, const uint32_t* __restrict__ pos_in,
                                                         uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out, long T, long V, int shift, int bits,
                                                         long tile, const uint32_t* __restrict__ hist) {
  __shared__ RankShared<256, TILE_BITS> s;
  static_assert(1 << TILE_BITS == 512, "two digits a thread");
  uint32_t all0 = 0, all1 = 0, earlier0 = 0, earlier1 = 0;
#pragma unroll 16
  for (int t = 0; t < (int)gridDim.x; ++t) {
    const uint2 c = reinterpret_cast<const uint2*>(hist + ((long)t << TILE_BITS))[threadIdx.x];
    all0 += c.x; all1 += c.y;
    if (t < (int)blockIdx.x) { earlier0 += c.x; earlier1 += c.y; }
  }
  s.base[2 * threadIdx.x] = all0;
  s.base[2 * threadIdx.x + 1] = all1;
  scan_digits(s);
  s.base[2 * threadIdx.x] += earlier0;
  s.base[2 * threadIdx.x + 1] += earlier1;
  __syncthreads();
  const long begin = blockIdx.x * tile, end = begin + tile < T ? begin + tile : T;
  for (long t = begin; t < end; t += TILE) place<256, TILE_BITS, TILE / 256, FIRST, false>(s, ids, V, key_in, pos_in, key_out, pos_out, t, end, shift, bits);
}

// ------------------------------------------------------------------------------------------------ sums of sorted rows
struct SumArgs {
  const void* dout;
  const uint32_t *key, *pos;
  void* dw;
  float* part;           // [chunks][2][pitch]: sums of a chunk's run that began in an earlier chunk (0), of one that goes on in the next (1)
  long T, V;
  int D, pitch, cp, lanes_log2, slices, accumulate;
  float scale;
};

template <bool OBF, int VEC>
__device__ __forceinline__ void finish_row(const SumArgs& a, uint32_t k, int c, float (&acc)[VEC]) {
  const long at = (long)k * a.D + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
  if (a.accumulate) {
    if constexpr (VEC == 4 && OBF) {   // 8 bytes of bfloat16
      const u32x2 w = *(glb<const u32x2>)((glb<const uint16_t>)a.dw + at);
      acc[0] += bf16_lo(w.x); acc[1] += bf16_hi(w.x); acc[2] += bf16_lo(w.y); acc[3] += bf16_hi(w.y);
    } else {
      float old[VEC];
      load_vec<OBF, VEC>(a.dw, at, old);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += old[i];
    }
  }
  store_vec<OBF, VEC>(a.dw, at, acc);
}

// `bytes` zeros from p (2-byte aligned) by `lanes` (8 or 64) lanes: 16 at a time between the aligned ends
__device__ __forceinline__ void zero_bytes(char* p, long bytes, int lane, int lanes) {
  long head = (16 - ((uintptr_t)p & 15)) & 15;
  if (head > bytes) head = bytes;
  if (lane * 2 < head) *(glb<uint16_t>)(p + lane * 2) = 0;
  const long wide = (bytes - head) / 16;
  for (long i = lane; i < wide; i += lanes) *(glb<u32x4>)(p + head + i * 16) = u32x4{0, 0, 0, 0};
  const long done = head + wide * 16;
  if (done + lane * 2 < bytes) *(glb<uint16_t>)(p + done + lane * 2) = 0;
}

// One group of `lanes` lanes sums the rows of `cp` consecutive sorted positions over lanes * VEC columns.  Workgroups behind those
// write zeros to the rows that have no position (found by bisection: the sorted classes are in L2).
constexpr int FILL_ROWS = 64;
template <bool IBF, bool OBF, int VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a, int sum_blocks) {
  if ((int)blockIdx.x >= sum_blocks) {
    __shared__ int absent[FILL_ROWS];
    for (long r0 = (long)((int)blockIdx.x - sum_blocks) * FILL_ROWS; r0 < a.V; r0 += (long)((int)gridDim.x - sum_blocks) * FILL_ROWS) {
      if (threadIdx.x < FILL_ROWS) {
        const long row = r0 + threadIdx.x;
        long lo = 0, hi = a.T;
        while (lo < hi) {
          const long mid = (lo + hi) >> 1;
          if ((long)a.key[mid] < row) lo = mid + 1;
          else hi = mid;
        }
        absent[threadIdx.x] = row < a.V && !(lo < a.T && (long)a.key[lo] == row);
      }
      __syncthreads();
      constexpr int ES = OBF ? 2 : 4;
      const int zl = a.D * ES <= 256 ? 8 : 64;      // short rows: eight lanes each
      for (int r = threadIdx.x / zl; r < FILL_ROWS; r += 256 / zl)
        if (absent[r]) zero_bytes(reinterpret_cast<char*>(a.dw) + (r0 + r) * a.D * ES, (long)a.D * ES, threadIdx.x & (zl - 1), zl);
      __syncthreads();
    }
    return;
  }
  const int lanes = 1 << a.lanes_log2;
  const long group = (long)blockIdx.x * (256 >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
  const long chunk = group / a.slices;
  const int c = ((int)(group - chunk * a.slices) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
  const long p0 = chunk * a.cp;
  if (p0 >= a.T || c >= a.D) return;
  const long p1 = p0 + a.cp < a.T ? p0 + a.cp : a.T;
  const uint32_t none = (uint32_t)a.V;
  const uint32_t before = p0 > 0 ? a.key[p0 - 1] : none, behind = p1 < a.T ? a.key[p1] : none;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  uint32_t cur = none;
  bool first = true;    // whether the current run is the chunk's first
  const auto flush = [&](bool last) {
    if (cur == none) return;
    if (first && cur == before) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a.part[(chunk * 2) * a.pitch + c + i] = acc[i];
    } else if (last && cur == behind) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a.part[(chunk * 2 + 1) * a.pitch + c + i] = acc[i];
    } else finish_row<OBF, VEC>(a, cur, c, acc);
  };
  constexpr int AHEAD = 8;
  for (long p = p0; p < p1; p += AHEAD) {
    uint32_t k[AHEAD];
    float v[AHEAD][VEC];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool in = p + u < p1;
      k[u] = in ? a.key[p + u] : none;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
      if (k[u] != none) load_vec<IBF, VEC>(a.dout, (long)a.pos[p + u] * a.D + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (p + u < p1 && k[u] != cur) {
        if (p + u > p0) { flush(false); first = false; }
        cur = k[u];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += v[u][i];
    }
  }
  flush(true);
}

// A run that goes on behind the chunk it began in: its first partial row plus those of the chunks that follow, shared over the groups of
// a workgroup and added up in a fixed order.
template <bool OBF, int VEC>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a, long chunks, long first) {      // chunks from `first` on
  const int lanes = 1 << a.lanes_log2, groups = 256 >> a.lanes_log2;
  const long chunk = first + blockIdx.x;
  const uint32_t none = (uint32_t)a.V;
  const long p0 = chunk * a.cp, p1 = p0 + a.cp;
  if (p1 >= a.T) return;
  const uint32_t k = a.key[p1 - 1];
  if (k == none || a.key[p1] != k) return;
  if (a.key[p0] == k && p0 > 0 && a.key[p0 - 1] == k) return;       // began earlier: joined there
  __shared__ float sums[256 * VEC];
  const int g = threadIdx.x >> a.lanes_log2, l = threadIdx.x & (lanes - 1);
  const int c = ((int)blockIdx.y * lanes + l) * VEC;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  if (c < a.D) {
    // eight chunks of this group at a time: their rows are read while it is not known yet whether they belong to the run
    constexpr int AHEAD = 8;
    bool on = true;
    for (long q = chunk + 1 + g; on && q < chunks; q += AHEAD * groups) {
      uint32_t key[AHEAD];
      float v[AHEAD][VEC];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const long x = q + u * groups;
        const long y = x < chunks ? x : q;
        key[u] = a.key[y * a.cp];
        load_vec<false, VEC>(a.part, (y * 2) * a.pitch + c, v[u]);
        if (x >= chunks) key[u] = none;
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        on = key[u] == k;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += on ? v[u][i] : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[i * 256 + threadIdx.x] = acc[i];
  __syncthreads();
  if (g == 0 && c < a.D) {
    float row[VEC];
    load_vec<false, VEC>(a.part, (chunk * 2 + 1) * a.pitch + c, row);
    for (int j = 0; j < groups; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) row[i] += sums[i * 256 + j * lanes + l];
    finish_row<OBF, VEC>(a, k, c, row);
  }
}

// ------------------------------------------------------------------------------------------------ small tables
// A table of few classes needs no sorting: every thread holds the sums of all classes over its VEC columns in LDS, [class][thread] -- free of bank
// conflicts whatever the classes are -- and walks its rows in order.  Class V is the bin of rows without one.  Sums begin with -0, which no
// addition tells from nothing: a sum that still is -0 at the end had no position (or only zeros of that sign).
// dW's value k from its sum
struct Target { void* dw; int bf16, accumulate; float scale; };
__device__ __forceinline__ void finish_value(const Target& t, long k, float sum) {
  const bool none = __float_as_uint(sum) == 0x80000000u;
  if (none && t.accumulate) return;
  const float s = none ? 0.f : sum * t.scale;
  if (t.bf16) {
    const glb<uint16_t> to = (glb<uint16_t>)t.dw + k;
    *to = to_bf16(t.accumulate ? bf16_lo(*to) + s : s);
  } else {
    const glb<float> to = (glb<float>)t.dw + k;
    *to = t.accumulate ? *to + s : s;
  }
}

struct SmallArgs {
  const void* dout; const int64_t* ids; float* part;       // part: [workgroups][V][D]
  long T, per;                                             // per: rows of a workgroup
  int V, D, lanes_log2, slices;
};
// VEC values as they lie in memory: float32, or bfloat16 by twos
template <bool IBF, int VEC> struct Raw { typedef float type __attribute__((ext_vector_type(VEC))); };
template <> struct Raw<true, 4> { typedef u32x2 type; };
template <> struct Raw<true, 2> { typedef uint32_t type; };
template <> struct Raw<true, 1> { typedef uint16_t type; };
template <bool IBF, int VEC>
__device__ __forceinline__ auto values_of(typename Raw<IBF, VEC>::type w) {
  typedef float vec __attribute__((ext_vector_type(VEC)));
  if constexpr (!IBF) return w;
  else if constexpr (VEC == 4) return vec{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
  else if constexpr (VEC == 2) return vec{bf16_lo(w), bf16_hi(w)};
  else return vec(bf16_lo(w));
}
template <bool IBF, int VEC>
__global__ __launch_bounds__(256) void embed_small_kernel(SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) float sums[];       // [V + 1][256][VEC]
  typedef float vec __attribute__((ext_vector_type(VEC)));
  typedef typename Raw<IBF, VEC>::type raw;
  vec* const mine = reinterpret_cast<vec*>(sums) + threadIdx.x;
  const int lanes = 1 << a.lanes_log2, streams = 256 >> a.lanes_log2;
  const long block = blockIdx.x / a.slices, r0 = block * a.per, r1 = r0 + a.per < a.T ? r0 + a.per : a.T;
  const int c = ((int)(blockIdx.x % a.slices) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
  for (int v = 0; v <= a.V; ++v) mine[v * 256] = vec(-0.f);
  constexpr int AHEAD = 8;
  if (c < a.D) {
    long id[AHEAD];
    raw x[AHEAD];
    const auto fetch = [&](long t0) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const long t = t0 + u * streams, r = t < r1 ? t : r1 - 1;
        id[u] = ((glb<const int64_t>)a.ids)[r];
        x[u] = *(glb<const raw>)((glb<const char>)a.dout + (r * a.D + c) * (IBF ? 2 : 4));
      }
      __builtin_amdgcn_sched_barrier(0);         // all of them on their way before the first is looked at
    };
    long t0 = r0 + (threadIdx.x >> a.lanes_log2);
    if (t0 < r1) fetch(t0);
    while (t0 < r1) {
      int now[AHEAD];
      raw y[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        now[u] = (t0 + u * streams < r1 && id[u] >= 0 && id[u] < a.V ? (int)id[u] : a.V) * 256;
        y[u] = x[u];
      }
      t0 += AHEAD * streams;
      if (t0 < r1) fetch(t0);
#pragma unroll
      for (int u = 0; u < AHEAD; u += 2) {       // two at a time, so that the second need not wait for the first's way through LDS
        const vec first = mine[now[u]] + values_of<IBF, VEC>(y[u]), second = mine[now[u + 1]];
        mine[now[u]] = first;
        mine[now[u + 1]] = (now[u] == now[u + 1] ? first : second) + values_of<IBF, VEC>(y[u + 1]);
      }
    }
  }
  __syncthreads();
  if (c >= a.D) return;
  const vec* const all = reinterpret_cast<const vec*>(sums) + (threadIdx.x & (lanes - 1));
#pragma unroll 4
  for (int v = threadIdx.x >> a.lanes_log2; v < a.V; v += streams) {
    vec sum = all[v * 256];
    for (int q = 1; q < streams; ++q) sum += all[v * 256 + q * lanes];
    *(glb<vec>)((glb<float>)a.part + (block * a.V + v) * a.D + c) = sum;
  }
}

// Few positions of a table that is not small: a workgroup takes 16 classes, up to `per` positions and 16 threads' columns.  It first lists those of its
// positions that have one of its classes -- in order, a wave's quarter after the other's --, then sums their rows as above, 16 streams of
// them.  No sorting, and no more than per / 16 rows in a thread's way whatever the classes are.
constexpr int RANGE = 16, RANGE_MOST = 1280, RANGE_LANES = 16;      // a list entry: 12 bits of the position, 4 of the class
template <bool IBF, int VEC>
__global__ __launch_bounds__(256) void embed_range_kernel(SmallArgs a, int groups, Target t) {
  extern __shared__ __attribute__((aligned(16))) float sums[];       // [RANGE + 1][256][VEC]
  __shared__ uint16_t list[RANGE_MOST];
  __shared__ int found[4];
  typedef float vec __attribute__((ext_vector_type(VEC)));
  typedef typename Raw<IBF, VEC>::type raw;
  vec* const mine = reinterpret_cast<vec*>(sums) + threadIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slice = blockIdx.x % a.slices, rest = blockIdx.x / a.slices, group = rest % groups;
  const long block = rest / groups, r0 = block * a.per;
  const int n = (int)(r0 + a.per < a.T ? a.per : a.T - r0), quarter = (n + 3) / 4, v0 = group * RANGE, most = a.V - v0 < RANGE ? a.V - v0 : RANGE;
  const int c = (slice * RANGE_LANES + (threadIdx.x & (RANGE_LANES - 1))) * VEC;
  {
    uint16_t* const own = list + wave * quarter;
    const int end = (wave + 1) * quarter < n ? (wave + 1) * quarter : n;
    int count = 0;
    constexpr int AHEAD = 4;
    for (int t0 = wave * quarter + lane; t0 - lane < end; t0 += 64 * AHEAD) {
      long id[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) id[u] = t0 + 64 * u < end ? ((glb<const int64_t>)a.ids)[r0 + t0 + 64 * u] : -1;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const bool in = id[u] >= v0 && id[u] < v0 + most;
        const uint64_t all = __ballot(in);
        if (in) own[count + __popcll(all & ((1ull << lane) - 1ull))] = (uint16_t)((t0 + 64 * u) << 4 | (int)(id[u] - v0));
        count += __popcll(all);
      }
    }
    if (lane == 0) found[wave] = count;
  }
  __syncthreads();
  const int f0 = found[0], f1 = f0 + found[1], f2 = f1 + found[2], total = f2 + found[3];
  constexpr int AHEAD = 8, STREAMS = 256 / RANGE_LANES;
  if (total) {
#pragma unroll
    for (int v = 0; v <= RANGE; ++v) mine[v * 256] = vec(-0.f);
  }
  for (int k0 = threadIdx.x / RANGE_LANES; c < a.D && k0 < total; k0 += AHEAD * STREAMS) {
    int at[AHEAD];
    raw x[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * STREAMS < total ? k0 + u * STREAMS : k0;
      const int w = (k >= f0) + (k >= f1) + (k >= f2), begin = w == 0 ? 0 : w == 1 ? f0 : w == 2 ? f1 : f2;
      const uint32_t entry = list[w * quarter + k - begin];
      at[u] = (k0 + u * STREAMS < total ? (int)(entry & 15u) : RANGE) * 256;
      x[u] = *(glb<const raw>)((glb<const char>)a.dout + ((r0 + (entry >> 4)) * a.D + c) * (IBF ? 2 : 4));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < AHEAD; u += 2) {
      const vec first = mine[at[u]] + values_of<IBF, VEC>(x[u]), second = mine[at[u + 1]];
      mine[at[u]] = first;
      mine[at[u + 1]] = (at[u] == at[u + 1] ? first : second) + values_of<IBF, VEC>(x[u + 1]);
    }
  }
  __syncthreads();
  const int v = threadIdx.x / RANGE_LANES;
  if (v >= most || c >= a.D) return;
  const vec* const all = reinterpret_cast<const vec*>(sums) + v * 256 + (threadIdx.x & (RANGE_LANES - 1));
  vec sum = vec(-0.f);
  if (total) {
#pragma unroll
    for (int q = 0; q < STREAMS; ++q) sum += all[q * RANGE_LANES];
  }
  if (t.dw) {                // the only part
#pragma unroll
    for (int k = 0; k < VEC; ++k) finish_value(t, (long)(v0 + v) * a.D + c + k, sum[k]);
  } else
    *(glb<vec>)((glb<float>)a.part + (block * a.V + v0 + v) * a.D + c) = sum;
}

// Q threads a value over the parts: 16, or 1 for few parts
template <int Q>
__global__ __launch_bounds__(1024) void embed_small_join_kernel(const float* __restrict__ part, int parts, long n, Target t) {
  constexpr int C = 1024 / Q;
  __shared__ float w[Q][C];
  const int c = threadIdx.x % C, q = threadIdx.x / C;
  const long k = (long)blockIdx.x * C + c;
  float s = -0.f;
  if (k < n) {
#pragma unroll 8
    for (int p = q; p < parts; p += Q) s += part[p * n + k];
  }
  if constexpr (Q > 1) {
    w[q][c] = s;
    __syncthreads();
  }
  if (q || k >= n) return;
  for (int p = 1; p < Q; ++p) s += w[p][c];
  finish_value(t, k, s);
}

__global__ __launch_bounds__(256) void embed_zero_kernel(uint16_t* __restrict__ p, long halves) {   // a gradient without positions
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < halves; i += (long)gridDim.x * 256) p[i] = 0;
}

constexpr long MOST_BLOCKS = 1L << 23;      // of 256 threads: a launch has fewer than 2^32 in a dimension

int log2_ceil(long x) { int l = 0; while ((1L << l) < x) ++l; return l; }

struct Layout { long tile, tiles, chunks; int cp, pitch, passes, bits; size_t key[2], pos[2], hist, part, total; };
Layout layout_of(long T, long V, long D) {
  Layout L;
  const int all = log2_ceil(V + 1);                           // keys are 0 .. V
  L.passes = cdiv(all, T <= ONE_TILE ? ONE_BITS : TILE_BITS);
  L.bits = cdiv(all, L.passes);
  L.tile = TILE * cdiv(T, (long)TILE * MAX_TILES);
  L.tiles = (T + L.tile - 1) / L.tile;
  // Positions of one chunk: 64 where that leaves the chip thousands of waves, fewer for small inputs, down to 8 (one round of loads).
  L.cp = 64;
  while (L.cp > 8 && T * D / L.cp < (1L << 21)) L.cp >>= 1;
  L.chunks = (T + L.cp - 1) / L.cp;
  L.pitch = (int)((D + 7) / 8 * 8);
  size_t at = 0;
  const auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  for (int i = 0; i < 2; ++i) { L.key[i] = take(4 * (size_t)T); L.pos[i] = take(4 * (size_t)T); }
  L.hist = take((size_t)L.tiles << (TILE_BITS + 2));
  L.part = take((size_t)L.chunks * 2 * L.pitch * 4);
  L.total = at;
  return L;
}

// The rule for small tables.  A thread takes as many columns (4, 2, 1) as leave its sums of all classes room in LDS.  Times in us, sorted and so:
// 2^20 x 64 bfloat16, 5 classes 129 and 34 (31 at a copy's rate); 65536 x 512 float32, 38 classes 49 and 32, 60 classes 48 and 40; 1000 x 16, 2 classes 15
// and 7.  One column a thread reads memory too slowly for large inputs (262144 x 128, 100 classes 61 and 56; 262144 x 512, 150 classes 189 and
// 246), and the parts of a large table take longer than its sorting (200 x 2048, 140 classes 16 and 26; 2000 x 2048, 60 classes 22 and 26).
struct SmallPlan { bool fits; int vec, lanes_log2, slices, blocks; long per; size_t lds, total; };
SmallPlan small_plan(long T, long V, long D, bool fours) {
  SmallPlan p{};
  const long room = 156 << 10;
  p.vec = 1;
  while (fours && p.vec < 4 && (V + 1) * 2048 * p.vec <= room) p.vec *= 2;
  p.fits = T >= 1 && (V + 1) * 1024 <= room && V * D <= (1L << 17) && (p.vec > 1 || V < 78 || T * D <= (1L << 25));
  if (!p.fits) return p;
  const long per_row = D / p.vec;
  p.lanes_log2 = log2_ceil(per_row) < 8 ? log2_ceil(per_row) : 8;
  p.slices = (int)((per_row + (1 << p.lanes_log2) - 1) >> p.lanes_log2);
  p.lds = (size_t)(V + 1) * 1024 * p.vec;
  long each = (160 << 10) / (long)p.lds;                     // workgroups of a CU
  each = each < 1 ? 1 : each > 8 ? 8 : each;
  // workgroups for the rows: their parts' way through memory (8 bytes a value, 4.6 TB/s) against the steps of a thread, 0.15 us each
  const double steps = (double)T / (256 >> p.lanes_log2);
  long blocks = (long)sqrt(0.15 * 4.6e6 * steps / (8.0 * V * D));
  if (blocks > 256 * each / p.slices) blocks = 256 * each / p.slices;
  if (blocks > (long)steps / 8) blocks = (long)steps / 8;
  if (blocks < 1) blocks = 1;
  p.per = (T + blocks - 1) / blocks;
  p.blocks = (int)((T + p.per - 1) / p.per);
  p.total = (size_t)p.blocks * V * D * 4;
  return p;
}
// embed_range_kernel: with no more positions than leave a workgroup 1280 when there are two workgroups a CU (72 KB of LDS), and no more than 2500
// workgroups.  Classes as a language has them / all positions in one class, float32, sorted and so, in us: 300 x 128, 1000 classes 18 / 17 and 6 / 8; 5003
// x 128, 1000 classes 24 / 26 and 14 / 21; 1000 x 256, 8000 classes 27 / 27 and 16 / 16.  With 2000 positions a workgroup: 4000 x 250, 1000
// classes 24 / 29 and 29 / 53; with 4000 workgroups: 1280 x 1000, 4000 classes 28 / 30 and 34 / 20.
struct RangePlan { bool fits; int vec, slices, groups, blocks; long per; size_t total; };
RangePlan range_plan(long T, long V, long D, bool fours) {
  RangePlan p{};
  if (T < 1) return p;
  p.vec = fours ? 4 : 1;
  p.slices = cdiv(D, RANGE_LANES * p.vec);
  p.groups = cdiv(V, RANGE);
  const long each = (long)p.slices * p.groups, room = 512 / each, most = room < 1 ? 1 : room;
  p.fits = T <= RANGE_MOST * most && each <= 2500;
  if (!p.fits) return p;
  long blocks = T / 256 < most ? T / 256 : most;            // 256 positions are not worth a part of their own
  if (blocks < 1) blocks = 1;
  p.per = (T + blocks - 1) / blocks;
  p.blocks = (int)((T + p.per - 1) / p.per);
  p.total = (size_t)p.blocks * V * D * 4;
  return p;
}
template <bool IBF, int VEC>
int launch_range(const SmallArgs& a, const RangePlan& p, const Target& t, hipStream_t st) {
  constexpr size_t LDS = (RANGE + 1) * 1024 * VEC;
  DPPM_TRY(lds_limit(reinterpret_cast<const void*>(embed_range_kernel<IBF, VEC>), LDS, "dppm_embedding_wgrad"));
  hipLaunchKernelGGL((embed_range_kernel<IBF, VEC>), dim3((unsigned)(p.blocks * p.groups * p.slices)), dim3(256), LDS, st, a, p.groups, p.blocks == 1 ? t : Target{});
  return DPPM_OK;
}

template <bool IBF, int VEC>
int launch_small(const SmallArgs& a, const SmallPlan& p, hipStream_t st) {
  DPPM_TRY(lds_limit(reinterpret_cast<const void*>(embed_small_kernel<IBF, VEC>), (int)p.lds, "dppm_embedding_wgrad"));
  hipLaunchKernelGGL((embed_small_kernel<IBF, VEC>), dim3((unsigned)(p.blocks * p.slices)), dim3(256), p.lds, st, a);
  return DPPM_OK;
}

template <bool IBF, bool OBF, int VEC>
void launch_sums(const SumArgs& s, long chunks, hipStream_t st) {
  const int per_block = 256 >> s.lanes_log2;
  const long sum_blocks = (chunks * s.slices + per_block - 1) / per_block;
  const long groups = (s.V + FILL_ROWS - 1) / FILL_ROWS, fill = s.accumulate ? 0 : groups < MOST_BLOCKS / 4 ? groups : MOST_BLOCKS / 4;
  hipLaunchKernelGGL((embed_sum_kernel<IBF, OBF, VEC>), dim3((unsigned)(sum_blocks + fill)), dim3(256), 0, st, s, (int)sum_blocks);
  for (long first = 0; first < chunks - 1; first += MOST_BLOCKS) {
    const long n = chunks - 1 - first < MOST_BLOCKS ? chunks - 1 - first : MOST_BLOCKS;
    hipLaunchKernelGGL((embed_join_kernel<OBF, VEC>), dim3((unsigned)n, (unsigned)s.slices), dim3(256), 0, st, s, chunks, first);
  }
}

}  // namespace
}  // namespace dppm

using namespace dppm;

#define DPPM_REQUIRE_TABLE(what)                                                                                                       \
  DPPM_REQUIRE(T >= 0 && V >= 1 && D >= 1, what ": T=%ld V=%ld D=%ld", (long)T, (long)V, (long)D);                                     \
  DPPM_REQUIRE(T < (1L << 31) && V < (1L << 31) && D <= (1L << 21), what ": T=%ld V=%ld D=%ld are too large", (long)T, (long)V, (long)D)

extern "C" int dppm_embedding_fwd(const void* weight, int bf16, const int64_t* ids, float scale, void* out, int64_t T, int64_t V, int64_t D,
                                  void* stream) {
  DPPM_REQUIRE_TABLE("dppm_embedding_fwd");
  if (T == 0) return DPPM_OK;
  DPPM_REQUIRE(weight && ids && out, "dppm_embedding_fwd: null pointer");
  const int vec = bf16 ? 8 : 4;
  // 16 bytes a lane where rows allow it; else one value a lane
  const bool wide = D % vec == 0 && ((uintptr_t)weight | (uintptr_t)out) % 16 == 0;
  const long per_row = wide ? D / vec : D;
  const int tl = log2_ceil(per_row) < 8 ? log2_ceil(per_row) : 8;
  const long rows = (256 >> tl) * FWD_ROWS, es = bf16 ? 2 : 4;
  const hipStream_t st = as_stream(stream);
  for (long t0 = 0; t0 < T; t0 += rows * MOST_BLOCKS) {
    const long n = T - t0 < rows * MOST_BLOCKS ? T - t0 : rows * MOST_BLOCKS;
    const dim3 grid((unsigned)((n + rows - 1) / rows)), block(256);
    const int64_t* const at = ids + t0;
    void* const to = reinterpret_cast<char*>(out) + t0 * D * es;
    if (bf16) {
      if (wide) hipLaunchKernelGGL((embed_fwd_kernel<true, 8>), grid, block, 0, st, weight, at, scale, to, n, (long)V, (int)D, tl);
      else hipLaunchKernelGGL((embed_fwd_kernel<true, 1>), grid, block, 0, st, weight, at, scale, to, n, (long)V, (int)D, tl);
    } else {
      if (wide) hipLaunchKernelGGL((embed_fwd_kernel<false, 4>), grid, block, 0, st, weight, at, scale, to, n, (long)V, (int)D, tl);
      else hipLaunchKernelGGL((embed_fwd_kernel<false, 1>), grid, block, 0, st, weight, at, scale, to, n, (long)V, (int)D, tl);
    }
  }
  return check_launch("dppm_embedding_fwd");
}

extern "C" size_t dppm_embedding_wgrad_workspace_bytes(int64_t T, int64_t V, int64_t D) {
  if (T < 1 || V < 1 || D < 1 || T >= (1L << 31) || V >= (1L << 31) || D > (1L << 21)) return 0;
  const size_t sorted = layout_of(T, V, D).total, ones = small_plan(T, V, D, false).total, fours = D % 4 == 0 ? small_plan(T, V, D, true).total : 0;
  const size_t ones_r = range_plan(T, V, D, false).total, fours_r = D % 4 == 0 ? range_plan(T, V, D, true).total : 0;
  size_t most = sorted;
  for (const size_t n : {ones, fours, ones_r, fours_r}) most = n > most ? n : most;
  return most;      // the largest, so that the size does not depend on types and addresses
}

extern "C" int dppm_embedding_wgrad(const void* dout, int dout_bf16, const int64_t* ids, float scale, void* dweight, int dweight_bf16, int accumulate,
                                    int64_t T, int64_t V, int64_t D, void* workspace, size_t workspace_bytes, void* stream) {
  DPPM_REQUIRE_TABLE("dppm_embedding_wgrad");
  DPPM_REQUIRE(dweight, "dppm_embedding_wgrad: null pointer");
  const hipStream_t st = as_stream(stream);
  if (T == 0) {
    if (!accumulate) {
      const long halves = V * D * (dweight_bf16 ? 1 : 2);
      const long blocks = (halves + 255) / 256;
      hipLaunchKernelGGL(embed_zero_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, reinterpret_cast<uint16_t*>(dweight), halves);
    }
    return check_launch("dppm_embedding_wgrad");
  }
  DPPM_REQUIRE(dout && ids && workspace, "dppm_embedding_wgrad: null pointer");
  const Layout L = layout_of(T, V, D);
  const size_t need = dppm_embedding_wgrad_workspace_bytes(T, V, D);
  DPPM_REQUIRE(workspace_bytes >= need, "dppm_embedding_wgrad: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  DPPM_REQUIRE((uintptr_t)workspace % 16 == 0, "dppm_embedding_wgrad: the workspace must be 16-byte aligned");
  char* ws = reinterpret_cast<char*>(workspace);
  const bool fours = D % 4 == 0 && (uintptr_t)dout % (dout_bf16 ? 8 : 16) == 0;
  const SmallPlan small = small_plan(T, V, D, fours);
  const RangePlan range = range_plan(T, V, D, fours);
  if (small.fits || range.fits) {
    SmallArgs a{dout, ids, reinterpret_cast<float*>(ws), (long)T, small.per, (int)V, (int)D, small.lanes_log2, small.slices};
    const Target t{dweight, dweight_bf16, accumulate, scale};
    int parts = small.blocks;
    if (small.fits) {
      if (dout_bf16) DPPM_TRY(small.vec == 4 ? (launch_small<true, 4>(a, small, st)) : small.vec == 2 ? (launch_small<true, 2>(a, small, st)) : (launch_small<true, 1>(a, small, st)));
      else DPPM_TRY(small.vec == 4 ? (launch_small<false, 4>(a, small, st)) : small.vec == 2 ? (launch_small<false, 2>(a, small, st)) : (launch_small<false, 1>(a, small, st)));
    } else {
      a.per = range.per; a.slices = range.slices;
      parts = range.blocks;
      if (dout_bf16) DPPM_TRY(range.vec == 4 ? (launch_range<true, 4>(a, range, t, st)) : (launch_range<true, 1>(a, range, t, st)));
      else DPPM_TRY(range.vec == 4 ? (launch_range<false, 4>(a, range, t, st)) : (launch_range<false, 1>(a, range, t, st)));
    }
    const long n = V * D;
    if (small.fits || parts > 1) {
      if (parts <= 8) hipLaunchKernelGGL((embed_small_join_kernel<1>), dim3((unsigned)((n + 1023) / 1024)), dim3(1024), 0, st, a.part, parts, n, t);
      else hipLaunchKernelGGL((embed_small_join_kernel<16>), dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, st, a.part, parts, n, t);
    }
    return check_launch("dppm_embedding_wgrad");
  }
  SortBufs b;
  for (int i = 0; i < 2; ++i) {
    b.key[i] = reinterpret_cast<uint32_t*>(ws + L.key[i]);
    b.pos[i] = reinterpret_cast<uint32_t*>(ws + L.pos[i]);
  }
  if (T <= ONE_TILE) {
    hipLaunchKernelGGL(sort_one_kernel, dim3(1), dim3(1024), 0, st, ids, (long)T, (long)V, L.passes, L.bits, b);
  } else {
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + L.hist);
    const dim3 grid((unsigned)L.tiles), block(256);
    for (int p = 0; p < L.passes; ++p) {
      const int in = (p + 1) & 1, out = p & 1;
      if (p == 0) {
        hipLaunchKernelGGL((sort_count_kernel<true>), grid, block, 0, st, ids, b.key[in], (long)T, (long)V, 0, L.bits, L.tile, hist);
        hipLaunchKernelGGL((sort_place_kernel<true>), grid, block, 0, st, ids, b.key[in], b.pos[in], b.key[out], b.pos[out], (long)T, (long)V, 0, L.bits, L.tile, hist);
      } else {
        hipLaunchKernelGGL((sort_count_kernel<false>), grid, block, 0, st, ids, b.key[in], (long)T, (long)V, L.bits * p, L.bits, L.tile, hist);
        hipLaunchKernelGGL((sort_place_kernel<false>), grid, block, 0, st, ids, b.key[in], b.pos[in], b.key[out], b.pos[out], (long)T, (long)V, L.bits * p, L.bits, L.tile, hist);
      }
    }
  }
  SumArgs s;
  s.dout = dout; s.key = b.key[(L.passes - 1) & 1]; s.pos = b.pos[(L.passes - 1) & 1]; s.dw = dweight;
  s.part = reinterpret_cast<float*>(ws + L.part);
  s.T = T; s.V = V; s.D = (int)D; s.pitch = L.pitch; s.cp = L.cp; s.accumulate = accumulate != 0; s.scale = scale;
  const int vec = dout_bf16 ? 8 : 4;
  const bool wide = D % vec == 0 && (uintptr_t)dout % 16 == 0 && (uintptr_t)dweight % 16 == 0;
  const long per_row = wide ? D / vec : D;
  s.lanes_log2 = log2_ceil(per_row) < 6 ? log2_ceil(per_row) : 6;
  s.slices = (int)((per_row + (1 << s.lanes_log2) - 1) >> s.lanes_log2);
  if (dout_bf16) {
    if (dweight_bf16) wide ? launch_sums<true, true, 8>(s, L.chunks, st) : launch_sums<true, true, 1>(s, L.chunks, st);
    else wide ? launch_sums<true, false, 8>(s, L.chunks, st) : launch_sums<true, false, 1>(s, L.chunks, st);
  } else {
    if (dweight_bf16) wide ? launch_sums<false, true, 4>(s, L.chunks, st) : launch_sums<false, true, 1>(s, L.chunks, st);
    else wide ? launch_sums<false, false, 4>(s, L.chunks, st) : launch_sums<false, false, 1>(s, L.chunks, st);
  }
  return check_launch("dppm_embedding_wgrad");
}

// Softmax cross entropy over many classes, from the last hidden layer and the classes' rows, with both gradients; the scores never reach
// memory.  For row t of x with class y_t, weight w_t and n = denom (default: the number of rows that have a class):
//
//   s_tv = x_t . W_v      lse_t = log sum_v exp s_tv      loss = sum_t w_t / n (lse_t - s_{t,y_t})
//   d_tv = (exp(s_tv - lse_t) - [v = y_t]) w_t / n        dx_t = sum_v d_tv W_v        dW_v = sum_t d_tv x_t
//
// A row whose class lies outside [0, V) has none: its loss and its gradient row are zero, and it adds nothing to dW.
//
// Three matrix products, each 2 T V D operations, and the exponentials between them:
//  * scores: tiles of s on the matrix cores; from the accumulators each strip of classes gives its maximum and its sum of exponentials per
//    row, and (with gradients) the exponentials relative to the strip's maximum, in half precision for bfloat16 inputs -- they lie in [0, 1], where
//    its 11 bits keep 2^-11 of each down to 2^-14 of the maximum and 2^-25 of the maximum below, so that the only rounding of d that counts
//    is its own -- and in float32 for float32;
//  * rows: lse, the rows' losses;
//  * turn: exponentials to n d, rounded once to the operands' type (bfloat16: the own class's entry without loss in dx, plan_of says why not in dW);
//  * dx = d W and dW = d^T x: W and d are read transposed from LDS where the contracted dimension is not the contiguous one; x, the smallest,
//    is transposed in memory, with zeros for rows that have no class.
// The exponentials held at a time are those of one block of rows, at most 2^30 (bfloat16) or 2^27 (float32) of them -- or 64 rows', where that is
// more (more than 2^21 float32 classes) --: memory does not grow with T.  Several blocks add up dW in float32.  Few classes go another way, in one pass (few_kernel).
#include "dppm_common.h"
#include "dppm_tngemm.h"

namespace dppm {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // round to nearest even (v_cvt_pk_bf16_f32)
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {   // round to nearest even
  typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, halfx2{(_Float16)lo, (_Float16)hi});
}
__device__ __forceinline__ float half_lo(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)w); }
__device__ __forceinline__ float half_hi(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }
__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ float from_bf16(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// exp x: for float32 inputs to the last bits; else by one multiplication and v_exp_f32, off by |x| 2^-24 and the instruction's own last bit,
// far under the rounding of bfloat16 results
template <bool F32>
__device__ __forceinline__ float exp_of(float x) { return F32 ? expf(x) : __expf(x); }

// plane `p` (0 hi, 1 mid, 2 lo) of a float32 value: each the nearest bfloat16 to what the planes before it leave
__device__ __forceinline__ void split3(float v, uint16_t (&out)[3]) {
  out[0] = to_bf16(v);
  float r = v - from_bf16(out[0]);
  out[1] = to_bf16(r);
  r = r - from_bf16(out[1]);
  out[2] = to_bf16(r);
  if (!(fabsf(v) <= 3.3e38f)) { out[1] = 0; out[2] = 0; }     // infinity and NaN (and what rounds to infinity) stand in the first plane alone
}

// Stores of what the kernel does not read again.  Buffers larger than the 256 MB that the last cache holds go past the L2, where they would only
// push operands out (bfloat16, 8192 x 131072 exponentials: scores 7.3 -> 6.8 ms); smaller ones are left for the next kernel to find
// (float32, 2047 x 20011: 0.87 ms with stores past the L2, 0.83 without).
template <class V>
__device__ __forceinline__ void store_out(V v, V* p, bool past) {
  if (past) __builtin_nontemporal_store(v, p);
  else *p = v;
}
constexpr size_t CACHED = 256u << 20;

// ------------------------------------------------------------------------------------------------ counting rows, losses
// Of up to COUNTED rows, or of a workgroup of rows_kernel; one workgroup puts them together in a fixed order.  (One workgroup over all rows took
// 0.28 ms to count a million and 1.3 ms to sum their losses.)
struct RowsPart { double loss; uint32_t rows, pad; };
constexpr long COUNTED = 4096;

// 1 / denom, or 1 / (the sum of all threads' rows) where none is given; all NT threads get it
template <int NT>
__device__ __forceinline__ float inverse_of(uint32_t rows, float denom) {
  __shared__ uint32_t w[NT / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) rows += __shfl_xor(rows, o, 64);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = rows;
  __syncthreads();
  uint32_t all = 0;
  for (int i = 0; i < NT / 64; ++i) all += w[i];
  return 1.f / (denom > 0.f ? denom : (float)(all ? all : 1u));
}
// a thread's share of the rows with a class, from the targets or from what workgroups counted
template <int NT>
__device__ __forceinline__ uint32_t rows_with_class(const int64_t* target, long T, long V) {
  uint32_t n = 0;
#pragma unroll 8
  for (int t = threadIdx.x; t < T; t += NT) n += target[t] >= 0 && target[t] < V;
  return n;
}
template <int NT>
__device__ __forceinline__ uint32_t rows_counted(const uint32_t* counts, int n) {
  uint32_t sum = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += NT) sum += counts[i];
  return sum;
}
__device__ __forceinline__ void count_rows(const int64_t* target, long T, long V, int part, uint32_t* counts) {    // 256 threads
  __shared__ uint32_t w[4];
  const long t0 = part * COUNTED;
  uint32_t sum = rows_with_class<256>(target + t0, T - t0 < COUNTED ? T - t0 : COUNTED, V);
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) counts[part] = w[0] + w[1] + w[2] + w[3];
}

struct LossArgs { const RowsPart* parts; int n; float denom; float* loss; };   // loss null: nothing to do

// The loss of all rows, by one workgroup, in float64 and a fixed order.  `inv`: 1 / n, or null where nothing needed it before.
template <int NT>
__device__ __forceinline__ void sum_loss(const LossArgs& a, const float* inv) {
  __shared__ double ws[NT / 64];
  __shared__ uint32_t wn[NT / 64];
  double s = 0.0;
  uint32_t n = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.n; i += NT) { s += a.parts[i].loss; n += a.parts[i].rows; }
#pragma unroll
  for (int o = 32; o; o >>= 1) { s += __shfl_xor(s, o, 64); n += __shfl_xor(n, o, 64); }
  if ((threadIdx.x & 63) == 0) { ws[threadIdx.x >> 6] = s; wn[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    uint32_t rows = 0;
    for (int i = 0; i < NT / 64; ++i) { all += ws[i]; rows += wn[i]; }
    *a.loss = (float)(all * (inv ? *inv : 1.f / (a.denom > 0.f ? a.denom : (float)(rows ? rows : 1u))));
  }
}

__global__ __launch_bounds__(1024) void loss_kernel(LossArgs a) { sum_loss<1024>(a, nullptr); }

// ------------------------------------------------------------------------------------------------ scores
struct ScoreOut {
  float2* stats;            // [strips][rows of the block]: (maximum, sum of exponentials relative to it)
  float* target_score;      // [rows]
  const int64_t* target;    // [rows]
  void* e;                  // exponentials [rows][pitch], or null
  long pitch;
  int V;
  bool past;                // e is larger than the caches
};

// m = class, n = row: a lane holds classes of one row per fragment, so that maxima and sums run inside lanes and then over four of them.
template <class T, bool F32>
__global__ __launch_bounds__(T::NT) void scores_kernel(TnArgs g, ScoreOut o) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int tm, tn;
  tn_tile_of(blockIdx.x, gridDim.x, g.tiles_m, g.tiles_n, tm, tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  tn_acc acc[T::MI][T::NI];
  tn_product<T, false, false>(g, lds, m0, n0, 0, g.ksteps * g.pairs, acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ms = m0 + (wave % T::WGM) * T::WM, ns = n0 + (wave / T::WGM) * T::WN;     // this wave's strip of classes, its rows
  const int strip = ms / T::WM, first = ms + (lane >> 4) * 4;                         // class of acc[0][.][0]
#pragma unroll
  for (int j = 0; j < T::NI; ++j) {
    const int n = ns + j * 16 + (lane & 15);
    if (ms + T::WM > o.V) {      // classes behind the last
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (first + i * 16 + k >= o.V) acc[i][j][k] = -INFINITY;
    }
    const int64_t y = n < g.N ? o.target[n] : -1;
    const bool here = y >= ms && y < ms + T::WM && y < o.V;
    if (__any(here)) {
      const int at = (int)(y - first);
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (here && at == i * 16 + k) o.target_score[n] = acc[i][j][k];
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < T::MI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, acc[i][j][k]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float ref = top == -INFINITY ? 0.f : top;      // a strip of nothing but -inf: exponentials of 0
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < T::MI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = exp_of<F32>(acc[i][j][k] - ref);
        acc[i][j][k] = e;
        sum += e;
      }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16 && n < g.N && ms < o.V) o.stats[(long)strip * g.N + n] = make_float2(top, sum);
  }
  if (o.e) {
#pragma unroll
    for (int j = 0; j < T::WN / 32; ++j) {
      if constexpr (F32)
        tn_rows<T>(lds, acc, j, [&](int row, int m, const float (&v)[8]) {
          const int n = ns + j * 32 + row, c = ms + m;
          if (n < g.N && c < o.pitch) {
            f32x4* p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(o.e) + (long)n * o.pitch + c);
            store_out(f32x4{v[0], v[1], v[2], v[3]}, p, o.past);
            store_out(f32x4{v[4], v[5], v[6], v[7]}, p + 1, o.past);
          }
        });
      else
        tn_rows16<T>(lds, acc, j, pack_half, [&](int row, int m, u32x4 w) {
          const int n = ns + j * 32 + row, c = ms + m;
          if (n < g.N && c < o.pitch) store_out(w, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(o.e) + (long)n * o.pitch + c), o.past);
        });
    }
  }
}

// ------------------------------------------------------------------------------------------------ rows
struct RowsArgs {
  const float2* stats; int strips, rows; const int64_t* target; long V; const float *target_score, *row_weight;
  float *lse, *row_loss;
  RowsPart* parts;          // one a workgroup
};

// ROWS rows a workgroup, NT / ROWS threads each over the strips: 32, so that a strip's line is read whole, or 2 for few rows.  Threads 0 ..
// ROWS - 1 get their row's loss times its weight, thread 0 the sum of them and how many have a class.
template <int NT, int ROWS>
__device__ __forceinline__ RowsPart reduce_rows(const RowsArgs& a) {
  constexpr int LANES = NT / ROWS, AHEAD = 8;
  __shared__ float2 part[LANES][ROWS];
  const int r = threadIdx.x % ROWS, q = threadIdx.x / ROWS, n = blockIdx.x * ROWS + r;
  const float2* __restrict__ stats = a.stats;
  const int strips = a.strips, rows = a.rows;
  float top = -INFINITY, sum = 0.f;
  if (n < rows) {
    for (int s0 = q; s0 < strips; s0 += AHEAD * LANES) {
      float2 x[AHEAD];
      float t = top;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int s = s0 + u * LANES;
        x[u] = s < strips ? stats[(long)s * rows + n] : make_float2(-INFINITY, 0.f);
        t = fmaxf(t, x[u].x);
      }
      sum = top == -INFINITY ? sum : sum * expf(top - t);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (x[u].y != 0.f) sum += x[u].x == -INFINITY ? x[u].y : x[u].y * expf(x[u].x - t);      // NaN scores leave no maximum behind, only a sum
      top = t;
    }
  }
  part[q][r] = make_float2(top, sum);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) {
    __syncthreads();
    if (q < o) {
      const float2 x = part[q][r], y = part[q + o][r];
      const float t = fmaxf(x.x, y.x);
      const float sx = x.y == 0.f || x.x == -INFINITY ? x.y : x.y * expf(x.x - t), sy = y.y == 0.f || y.x == -INFINITY ? y.y : y.y * expf(y.x - t);
      part[q][r] = make_float2(t, sx + sy);
    }
  }
  RowsPart mine{0.0, 0u, 0u};
  if (q == 0 && n < rows) {
    const float t = part[0][r].x, s = part[0][r].y;
    const float l = t + logf(s);
    a.lse[n] = l;
    const int64_t y = a.target[n];
    const bool counts = y >= 0 && y < a.V;
    const float loss = counts ? l - a.target_score[n] : 0.f;
    a.row_loss[n] = loss;
    mine.rows = counts;
    if (loss != 0.f) mine.loss = (double)loss * (a.row_weight ? a.row_weight[n] : 1.f);      // rows without a class have 0, whatever their weight
  }
#pragma unroll
  for (int o = ROWS / 2; o; o >>= 1) { mine.loss += __shfl_xor(mine.loss, o, 64); mine.rows += __shfl_xor(mine.rows, o, 64); }
  return mine;
}

// counts not null: one more workgroup, which puts them together
template <int ROWS>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a, const uint32_t* __restrict__ counts, int n, float denom, float* __restrict__ inv) {
  if (counts && blockIdx.x == gridDim.x - 1) {
    const float x = inverse_of<256>(denom > 0.f ? 0u : rows_counted<256>(counts, n), denom);
    if (threadIdx.x == 0) *inv = x;
    return;
  }
  const RowsPart part = reduce_rows<256, ROWS>(a);
  if (threadIdx.x == 0) a.parts[blockIdx.x] = part;
}

// Up to 8 rows and no gradients: rows and loss by one workgroup with 128 threads a row, which spares a launch (for 5 rows against 32768 classes;
// with 32 threads a row, for up to 32 rows, it took 4 us longer than two launches)
__global__ __launch_bounds__(1024) void rows_and_loss_kernel(RowsArgs a, float denom, float* __restrict__ loss) {
  const RowsPart all = reduce_rows<1024, 8>(a);
  if (threadIdx.x == 0) *loss = (float)(all.loss * (1.f / (denom > 0.f ? denom : (float)(all.rows ? all.rows : 1u))));
}

// ------------------------------------------------------------------------------------------------ turn
struct TurnArgs {
  const void* e; long pitch;             // exponentials [rows][pitch]
  const float2* stats; const float* lse; const float* target_score; const int64_t* target; const float* row_weight; const float* inv;
  float* residual;                       // [rows], P == 1: what the row's own entry lost to bfloat16
  uint16_t* d; long plane;               // [planes][rows, whole tiles of 64][pitch]; in e's place for bfloat16
  int rows, whole, V, strip, across;     // whole: rows, to whole tiles of 64; strip: classes that share a maximum; across: workgroups for the classes
  bool past;                             // d is larger than the caches
};

// 16 rows x 512 classes a workgroup -- or, where the pitch is 64, 128 rows x 64 --, 8 classes a thread and row: n d_tv = e_tv * exp(max_strip - lse_t)
// * w_t, the row's own class from its float32 score.  1 / n is left to the gradients' float32 sums: without weights, the own entry of a class that is
// not yet likely is then next to -1 and loses nothing in bfloat16.  Rows behind the last (to whole tiles of 64) and without a class are zeros; so are
// classes behind the last, to the pitch.  P planes of d: 3 for float32; 1 for bfloat16, or 2 for few rows (plan_of).  LANES: threads a row.
template <bool F32, int P, int LANES>
__global__ __launch_bounds__(256) void turn_kernel(TurnArgs a, LossArgs l) {
  if (blockIdx.x == 0) {                  // one more workgroup, which sums the loss, with the last block of rows
    if (l.loss) sum_loss<256>(l, a.inv);
    return;
  }
  constexpr int ROWS = 1024 / LANES, GROUPS = LANES / 4;
  __shared__ float factor[GROUPS][ROWS + 1];     // of each 32 classes: strips of 32 are the shortest
  __shared__ float own[ROWS];
  __shared__ int at[ROWS];
  const int v0 = (blockIdx.x - 1) % a.across * (8 * LANES), t0 = (blockIdx.x - 1) / a.across * ROWS;
  {
    const int r = threadIdx.x % ROWS, k = threadIdx.x / ROWS, t = t0 + r, v = v0 + 32 * k;
    float f = 0.f, mine = 0.f;
    int where = -1;
    if (t < a.rows) {
      const int64_t y = a.target[t];
      if (y >= 0 && y < a.V) {
        const float g = a.row_weight ? a.row_weight[t] : 1.f;
        if (v < a.V) f = expf(a.stats[(long)(v / a.strip) * a.rows + t].x - a.lse[t]) * g;
        where = (int)y;
        if (k == 0) mine = (expf(a.target_score[t] - a.lse[t]) - 1.f) * g;
      }
    }
    factor[k][r] = f;
    if (k == 0) { own[r] = mine; at[r] = where; }
    if (P == 1 && k == 0 && v0 == 0 && t < a.rows) a.residual[t] = mine - from_bf16(to_bf16(mine));
  }
  __syncthreads();
  const int c = threadIdx.x % LANES * 8, v = v0 + c;
  if (v >= a.pitch) return;
#pragma unroll
  for (int r = threadIdx.x / LANES; r < ROWS; r += 256 / LANES) {
    const int t = t0 + r;
    if (t >= a.whole) return;
    const long to = (long)t * a.pitch + v;
    const float f = factor[c >> 5][r];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t < a.rows && f != 0.f) {
      if (F32) {
        const f32x4* e = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.e) + to);
        const f32x4 w0 = e[0], w1 = e[1];
        x[0] = w0.x; x[1] = w0.y; x[2] = w0.z; x[3] = w0.w; x[4] = w1.x; x[5] = w1.y; x[6] = w1.z; x[7] = w1.w;
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.e) + to);
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[2 * k] = half_lo(w[k]); x[2 * k + 1] = half_hi(w[k]); }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= f;
    }
    const int y = at[r] - v;
    if (y >= 0 && y < 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (y == k) x[k] = own[r];
    }
    if (P > 1) {
      uint16_t s[8][3];
#pragma unroll
      for (int k = 0; k < 8; ++k) split3(x[k], s[k]);
#pragma unroll
      for (int p = 0; p < P; ++p)
        store_out(u32x4{s[0][p] | (uint32_t)s[1][p] << 16, s[2][p] | (uint32_t)s[3][p] << 16, s[4][p] | (uint32_t)s[5][p] << 16, s[6][p] | (uint32_t)s[7][p] << 16},
                  reinterpret_cast<u32x4*>(a.d + p * a.plane + to), a.past);
    } else
      store_out(u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])}, reinterpret_cast<u32x4*>(a.d + to), a.past);
  }
}

// ------------------------------------------------------------------------------------------------ operands
// [rows][cols] of the caller, contiguous -> bfloat16 planes, as they stand [rows][pitch] (cols .. pitch zero) and/or transposed [cols][pitch_t]
// (rows .. pitch_t zero).  target, V (or null): rows without a class are zeros.  64 x 64 a workgroup.
struct LayOut {
  const void* src; int rows, cols;
  uint16_t* as_is; long pitch, plane;
  uint16_t* turned; long pitch_t, plane_t;
  const int64_t* target; long V;
  int across, wide;      // tiles across; wide: cols and the source's address allow 16-byte reads (4 or 8 values)
};

template <bool F32, bool WIDE>
__device__ __forceinline__ void lay_out_tile(const LayOut& a, int id) {
  const void* src = a.src;
  const int rows = a.rows, cols = a.cols;
  uint16_t *as_is = a.as_is, *turned = a.turned;
  const long pitch = a.pitch, plane = a.plane, pitch_t = a.pitch_t, plane_t = a.plane_t, V = a.V;
  const int64_t* target = a.target;
  constexpr int P = F32 ? 3 : 1, VEC = WIDE ? (F32 ? 4 : 8) : 1, PER_ROW = 64 / VEC;
  __shared__ uint16_t tile[P][64][66];
  const int c0 = id % a.across * 64, r0 = id / a.across * 64;
#pragma unroll 4
  for (int i = threadIdx.x; i < 64 * PER_ROW; i += 256) {
    const int r = i / PER_ROW, c = i % PER_ROW * VEC;
    uint16_t s[VEC][3];
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k][0] = s[k][1] = s[k][2] = 0;
    if (r0 + r < rows && c0 + c < cols && (!target || (target[r0 + r] >= 0 && target[r0 + r] < V))) {
      const long at = (long)(r0 + r) * cols + c0 + c;
      if constexpr (F32) {
        float v[VEC];
        if constexpr (WIDE) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(src) + at);
          v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        } else v[0] = reinterpret_cast<const float*>(src)[at];
#pragma unroll
        for (int k = 0; k < VEC; ++k) split3(v[k], s[k]);
      } else if constexpr (WIDE) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(src) + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) { s[2 * k][0] = (uint16_t)w[k]; s[2 * k + 1][0] = (uint16_t)(w[k] >> 16); }
      } else s[0][0] = reinterpret_cast<const uint16_t*>(src)[at];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (as_is && r0 + r < rows && c0 + c < pitch) {
        uint16_t* to = as_is + p * plane + (long)(r0 + r) * pitch + c0 + c;
        if constexpr (VEC == 8) *reinterpret_cast<u32x4*>(to) = u32x4{s[0][p] | (uint32_t)s[1][p] << 16, s[2][p] | (uint32_t)s[3][p] << 16,
                                                                     s[4][p] | (uint32_t)s[5][p] << 16, s[6][p] | (uint32_t)s[7][p] << 16};
        else if constexpr (VEC == 4) *reinterpret_cast<u32x2*>(to) = u32x2{s[0][p] | (uint32_t)s[1][p] << 16, s[2][p] | (uint32_t)s[3][p] << 16};
        else *to = s[0][p];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) tile[p][r][c + k] = s[k][p];
    }
  }
  if (!turned) return;
  __syncthreads();
  const int r = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int p = 0; p < P; ++p)
    for (int c = threadIdx.x >> 3; c < 64; c += 32) {
      if (c0 + c >= cols || r0 + r >= pitch_t) continue;
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = (uint32_t)tile[p][r + 2 * k][c] | ((uint32_t)tile[p][r + 2 * k + 1][c] << 16);
      *reinterpret_cast<u32x4*>(turned + p * plane_t + (long)(c0 + c) * pitch_t + r0 + r) = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// Everything that can be laid out before the products, in one launch: `first` workgroups for a, `second` for b, and the rest count the rows that have a
// class, COUNTED rows each (rows_kernel puts the counts together).
template <bool F32>
__global__ __launch_bounds__(256) void prepare_kernel(LayOut a, int first, LayOut b, int second, const int64_t* __restrict__ target, long T, long V,
                                                      uint32_t* __restrict__ counts) {
  const int id = blockIdx.x;
  if (id < first) {
    if (a.wide) lay_out_tile<F32, true>(a, id);
    else lay_out_tile<F32, false>(a, id);
  } else if (id < first + second) {
    if (b.wide) lay_out_tile<F32, true>(b, id - first);
    else lay_out_tile<F32, false>(b, id - first);
  } else
    count_rows(target, T, V, id - first - second, counts);
}

// ------------------------------------------------------------------------------------------------ gradients
struct GradOut {
  void* c; long ldc;          // [N][ldc], M values a row
  const float* add;           // float32 [N][ldc] that is added first, or null
  float* part; long part_stride;   // with splits: float32 [splits][N][ldc] instead
  const float* scale;         // what the products are multiplied with
  const int64_t* target;                 // dx: the rows' classes
  const float* residual;                 // dx, one plane of d: += residual[n] * A's row of target[n]; or null
  int c_bf16, past, wide;     // past: c is larger than the caches; wide: rows of c start on 16 bytes and M is a multiple of 8
};

__device__ __forceinline__ void put8(const GradOut& o, long at, int left, const float (&v)[8]) {
  if (o.c_bf16) {
    uint16_t* p = reinterpret_cast<uint16_t*>(o.c) + at;
    if (o.wide) store_out(u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])}, reinterpret_cast<u32x4*>(p), o.past);
    else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) p[k] = to_bf16(v[k]);
    }
  } else {
    float* p = reinterpret_cast<float*>(o.c) + at;
    if (o.wide) {
      reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) p[k] = v[k];
    }
  }
}

template <class T, bool TRA, bool TRB>
__device__ __forceinline__ void grad_tile(const TnArgs& g, const GradOut& o, char* lds, int id) {
  const int tiles = g.tiles_m * g.tiles_n, split = id / tiles;
  int tm, tn;
  tn_tile_of(id - split * tiles, tiles, g.tiles_m, g.tiles_n, tm, tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  const long steps = (long)g.ksteps * g.pairs;
  tn_acc acc[T::MI][T::NI];
  tn_product<T, TRA, TRB>(g, lds, m0, n0, (int)(steps * split / g.splits), (int)(steps * (split + 1) / g.splits), acc);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (TRA && o.residual && split == 0) {
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int n = n0 + (wave / T::WGM) * T::WN + 16 * j + (lane & 15), m = m0 + (wave % T::WGM) * T::WM + 4 * (lane >> 4);
      const float r = n < g.N ? o.residual[n] : 0.f;
      const uint16_t* row = g.A + (r != 0.f ? o.target[n] : 0) * g.lda + m;
      if (r != 0.f) {
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
          if (m + 16 * i < g.M) {        // a row's pitch is a multiple of 64
            const u32x2 w = *reinterpret_cast<const u32x2*>(row + 16 * i);
            acc[i][j] += r * tn_acc{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
          }
      }
    }
  }
  const float scale = *o.scale;
#pragma unroll
  for (int j = 0; j < T::NI; ++j) {
    bool has = true;
    if (TRA) {      // a row without a class has zeros in d, and in dx also where the table holds infinity or NaN
      const int n = n0 + (wave / T::WGM) * T::WN + 16 * j + (lane & 15);
      const int64_t y = o.target[n < g.N ? n : g.N - 1];
      has = y >= 0 && y < g.K;
    }
#pragma unroll
    for (int i = 0; i < T::MI; ++i) acc[i][j] = has ? acc[i][j] * scale : tn_acc{0.f, 0.f, 0.f, 0.f};
  }
  const int ms = m0 + (wave % T::WGM) * T::WM, ns = n0 + (wave / T::WGM) * T::WN;
  if (o.c_bf16 && o.wide && !o.part && !o.add) {
#pragma unroll
    for (int j = 0; j < T::WN / 32; ++j)
      tn_rows16<T>(lds, acc, j, pack_bf16, [&](int row, int m, u32x4 w) {
        const int n = ns + j * 32 + row;
        if (n < g.N && ms + m < g.M) store_out(w, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(o.c) + (long)n * o.ldc + ms + m), o.past);
      });
    return;
  }
#pragma unroll
  for (int j = 0; j < T::WN / 32; ++j)
    tn_rows<T>(lds, acc, j, [&](int row, int m, const float (&v)[8]) {
      const int n = ns + j * 32 + row, left = g.M - (ms + m);
      if (n >= g.N || left <= 0) return;
      const long at = (long)n * o.ldc + ms + m;
      GradOut q = o;
      if (o.part) {
        q.c = o.part + split * o.part_stride;
        q.c_bf16 = 0;
        q.wide = o.ldc % 4 == 0 && left >= 8;
        put8(q, at, left, v);
      } else if (o.add) {
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = v[k] + (k < left ? o.add[at + k] : 0.f);
        put8(q, at, left, w);
      } else put8(q, at, left, v);
    });
}

// Both gradients in one launch: few tiles of one leave room for the other's, and the last round of tiles is one and not two (the whole loss, bfloat16:
// 300 x 64, 100 classes 35.8 -> 28.8 us, 1000 x 256, 5000 classes 70 -> 57, 4099 x 1000, 50001 classes 1510 -> 1419).  The product with the
// longer tiles comes first.
struct GradJob { TnArgs g; GradOut o; };
template <class T>
__global__ __launch_bounds__(T::NT) void grad_kernel(GradJob x, GradJob w, int first, int w_first) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const bool early = (int)blockIdx.x < first;
  const int id = early ? blockIdx.x : blockIdx.x - first;
  if (early == (w_first != 0)) grad_tile<T, false, true>(w.g, w.o, lds, id);
  else grad_tile<T, true, false>(x.g, x.o, lds, id);
}

// The parts of a split product, in order, behind what was there before.
struct PartsJob { const float* part; long n; int splits; const float* add; void* c; int c_bf16; };
__global__ __launch_bounds__(256) void parts_kernel(PartsJob x, PartsJob w, int first) {
  const bool early = (int)blockIdx.x < first;
  const PartsJob& a = early ? x : w;
  const long at = early ? blockIdx.x : blockIdx.x - first, of = early ? first : gridDim.x - first;
  for (long i = at * 256 + threadIdx.x; i < a.n; i += of * 256) {
    float s = a.add ? a.add[i] : 0.f;
#pragma unroll 8
    for (int k = 0; k < a.splits; ++k) s += a.part[k * a.n + i];
    if (a.c_bf16) reinterpret_cast<uint16_t*>(a.c)[i] = to_bf16(s);
    else reinterpret_cast<float*>(a.c)[i] = s;
  }
}

// ------------------------------------------------------------------------------------------------ few classes
// Up to 16 classes of 512 values, 32 of 256, 64 of 128, 128 of 64 (of wider rows in two passes, below): all of W lies in LDS and a row's scores in the registers of four lanes, so that
// one pass over x gives the losses, dx and each workgroup's part of dW, and neither scores nor d reach memory.  x is read twice (the second
// time from the caches), dx written once.  A wave takes 16 rows at a time, in three products on the matrix cores:
//   s = W x^T    k = dims: lane i + 16 g holds row i, dims 32 step + 8 g .. + 7 (16 or 32 bytes of x); out come classes 4 g .. 4 g + 3 of row i,
//   dx^T = W^T d k = classes: those four are the operand as they stand; out come the same dims of row i as were read,
//   dW += d x    k = rows: d turned in LDS, x read again with a lane's four dims of row 4 t + g.
// float32: all three by v_mfma_f32_16x16x4_f32, 96 operations a value with the classes padded to 16.  bfloat16: scores in one exact product
// of the operands, dx with d in two bfloat16 planes, which hold 2^-17 of it; dW in float32 as well, its operands being a row's dims and not a dim's rows.
// LDS holds W twice, in the order of each product's fragments; slot 2 step + u, place q holds dim 32 step + 8 (q / 4) + 4 u + q % 4.
struct FewArgs {
  const void *x, *weight; const int64_t* target; const float* row_weight;
  const uint32_t* counts; int counters;            // 0: every workgroup counts for itself
  long T; int V, D; float denom;
  float* row_loss; void* dx;                       // dx null: losses only
  float* part; RowsPart* parts;                    // [workgroups][V][D], [workgroups]
  float* d; int slices;                            // in two passes: [T][padded classes]; slices of the dims
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
constexpr int FEW_CLASSES = 128, FEW_VALUES = 512;  // (padded classes / 16) * padded D at most FEW_VALUES: dW fits in 128 registers

// N (4 or 8) values of a row of D from dim d on, zeros behind the last (with N = 4 and WIDE, the caller sees to that): float32 as they are, bfloat16 by
// twos.  WIDE: D is a multiple of 8 and rows are aligned to 16 bytes.
template <bool F32, int N> struct Few;
template <int N> struct Few<true, N> { float v[N]; };
template <int N> struct Few<false, N> { uint32_t v[N / 2]; };
template <bool F32, bool WIDE, int N>
__device__ __forceinline__ Few<F32, N> load_few(const void* x, long row, int d, int D) {
  Few<F32, N> r;
  if constexpr (WIDE) {
    const long at = row * D + (d < D ? d : 0);
    if constexpr (F32) {
      const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(x) + at);
#pragma unroll
      for (int h = 0; h < N / 4; ++h) {
        const f32x4 w = p[h];
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[4 * h + e] = w[e];
      }
    } else if constexpr (N == 8) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(x) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.v[e] = w[e];
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint16_t*>(x) + at);
      r.v[0] = w.x;
      r.v[1] = w.y;
    }
    if (N == 8 && d >= D) r = Few<F32, N>{};
  } else {
    const long at = row * D;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int k = d + e < D ? d + e : 0;
      if constexpr (F32) {
        const float w = reinterpret_cast<const float*>(x)[at + k];
        r.v[e] = d + e < D ? w : 0.f;
      } else {
        const uint32_t w = d + e < D ? reinterpret_cast<const uint16_t*>(x)[at + k] : 0u;
        r.v[e / 2] = e & 1 ? r.v[e / 2] | w << 16 : w;
      }
    }
  }
  return r;
}

// CT: sixteens of classes, NC: sixty-fours of dims.  Wider rows go in two passes of this kernel: SCORES, whose W has all dims (and one order), leaves d in
// memory, 64 bytes a row and sixteen classes; GRADIENTS takes a slice of 64 NC dims of x and W a workgroup.
enum FewPass { ALL, SCORES, GRADIENTS };
template <bool F32, bool WIDE, int CT, int NC, FewPass PASS>
__global__ __launch_bounds__(256, PASS == SCORES ? 2 : CT * NC <= 2 ? 4 : CT == 8 ? 1 : 2) void few_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ __attribute__((aligned(16))) float turned[4][CT][16][20];
  __shared__ RowsPart sums[4];
  float* const wk = reinterpret_cast<float*>(lds);       // float32: [slot][ct][class][q]
  float* const wc = wk + (PASS == ALL ? NC * CT * 1024 : 0);     //  [slot][ct][q][class]
  uint16_t* const hk = reinterpret_cast<uint16_t*>(lds); // bfloat16: [step][ct][class][dim]
  uint16_t* const hc = hk + (PASS == ALL ? NC * CT * 1024 : 0);  //   [slot][q][class / 4][ct][class % 4]
  const int sixty_fours = PASS == SCORES ? (a.D + 127) / 128 * 2 : NC;
  const int slices = PASS == GRADIENTS ? a.slices : 1, block = blockIdx.x / slices, blocks = gridDim.x / slices, d0 = (blockIdx.x - block * slices) * 64 * NC;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  for (int k = threadIdx.x; k < 16 * CT * 8 * sixty_fours; k += 256) {
    const int v = k / (8 * sixty_fours), d = k % (8 * sixty_fours) * 8, st = d / 32, o = d % 32 / 8, ct = v / 16, c = v % 16;
    const Few<F32, 8> w = load_few<F32, WIDE, 8>(a.weight, v < a.V ? v : 0, v < a.V ? d0 + d : a.D, a.D);
    if constexpr (F32) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = (2 * st + u) * CT + ct;
        if (PASS != GRADIENTS) *reinterpret_cast<f32x4*>(wk + (at * 16 + c) * 16 + 4 * o) = f32x4{w.v[4 * u], w.v[4 * u + 1], w.v[4 * u + 2], w.v[4 * u + 3]};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (PASS != SCORES) wc[(at * 16 + 4 * o + e) * 16 + c] = w.v[4 * u + e];
      }
    } else {
      if (PASS != GRADIENTS) *reinterpret_cast<u32x4*>(hk + ((st * CT + ct) * 16 + c) * 32 + 8 * o) = u32x4{w.v[0], w.v[1], w.v[2], w.v[3]};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (PASS != SCORES) hc[((((2 * st + e / 4) * 16 + 4 * o + e % 4) * 4 + c / 4) * CT + ct) * 4 + c % 4] = (uint16_t)(w.v[e / 2] >> e % 2 * 16);
    }
  }
  float inv = 0.f;
  if (PASS != GRADIENTS && a.dx)
    inv = inverse_of<256>(a.denom > 0.f ? 0u : a.counters ? rows_counted<256>(a.counts, a.counters) : rows_with_class<256>(a.target, a.T, a.V), a.denom);
  __syncthreads();

  f32x4 dw[CT][NC][4];                                   // classes 4 g .. + 3 of dim 64 c + 4 i + e
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) dw[ct][c][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  RowsPart mine{0.0, 0u, 0u};
  constexpr int AHEAD = (NC == 1 && PASS == ALL) || !WIDE ? 2 : 4;                 // steps of 32 dims that are read together
  const int steps = (a.D - d0 < 64 * NC ? a.D - d0 + 31 : 64 * NC) / 32;
  for (long t0 = ((long)block * 4 + wave) * 16; t0 < a.T; t0 += (long)blocks * 64) {
    const long t = t0 + i < a.T ? t0 + i : a.T - 1;      // rows behind the last repeat it and count for nothing
    const int64_t y = a.target[t];
    const bool in = t0 + i < a.T, counts = in && y >= 0 && y < a.V;
    f32x4 p[CT];                                         // exponentials, then d
    if constexpr (PASS != GRADIENTS) {
      f32x4 s[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; 32 * s0 < a.D; s0 += AHEAD) {
        Few<F32, 8> v[AHEAD];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) v[h] = load_few<F32, WIDE, 8>(a.x, t, 32 * (s0 + h) + 8 * g, a.D);
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
          if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int ct = 0; ct < CT; ++ct) {
                const f32x4 w = *reinterpret_cast<const f32x4*>(wk + (((2 * (s0 + h) + u) * CT + ct) * 16 + i) * 16 + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e], v[h].v[4 * u + e], s[ct], 0, 0, 0);
              }
          } else {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              s[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const tn_frag*>(hk + (((s0 + h) * CT + ct) * 16 + i) * 32 + 8 * g),
                                                              __builtin_bit_cast(tn_frag, v[h]), s[ct], 0, 0, 0);
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (16 * ct + 4 * g + j < a.V) top = fmaxf(top, s[ct][j]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      float sum = 0.f, own = 0.f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int v = 16 * ct + 4 * g + j;
          p[ct][j] = v < a.V ? exp_of<F32>(s[ct][j] - top) : 0.f;
          sum += p[ct][j];
          if (v == y) own = s[ct][j];
        }
      sum += __shfl_xor(sum, 16, 64);
      own += __shfl_xor(own, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      own += __shfl_xor(own, 32, 64);
      const float loss = counts ? top + logf(sum) - own : 0.f;
      const float weight = counts && a.row_weight ? a.row_weight[t] : 1.f;
      if (g == 0) {
        if (in) a.row_loss[t] = loss;
        if (counts) { mine.rows += 1; mine.loss += loss != 0.f ? (double)loss * weight : 0.0; }
      }
      if (!a.dx) continue;

      const float share = weight * inv, r = 1.f / sum;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[ct][j] = counts ? (p[ct][j] * r - (16 * ct + 4 * g + j == y ? 1.f : 0.f)) * share : 0.f;      // d
    } else {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) p[ct] = in ? *reinterpret_cast<const f32x4*>(a.d + (t * CT + ct) * 16 + 4 * g) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (PASS == SCORES) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        if (in) *reinterpret_cast<f32x4*>(a.d + (t * CT + ct) * 16 + 4 * g) = p[ct];
      continue;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<f32x4*>(&turned[wave][ct][i][4 * g]) = p[ct];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    constexpr int PAIRS = (CT + 1) / 2;
    u32x4 plane[2][PAIRS];      // bfloat16: d in two planes, class 4 g + j of each sixteen, by pairs of sixteens
    if (!F32) {
      f32x4 rest[CT];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int ct = 0; ct < 2 * PAIRS; ++ct)
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t w = 0;
            if (ct < CT) {
              const float lo = k ? rest[ct][j] : p[ct][j], hi = k ? rest[ct][j + 1] : p[ct][j + 1];
              w = pack_bf16(lo, hi);
              if (k == 0) { rest[ct][j] = lo - __uint_as_float(w << 16); rest[ct][j + 1] = hi - __uint_as_float(w & 0xffff0000u); }
            }
            plane[k][ct / 2][2 * (ct & 1) + j / 2] = w;
          }
    }
#pragma unroll 1
    for (int st = 0; st < steps; ++st) {
      f32x4 o[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (!F32) {
          const uint16_t* w = hc + (((2 * st + u) * 16 + i) * 4 + g) * CT * 4;
#pragma unroll
          for (int k = 1; k >= 0; --k) {
            if constexpr (CT == 1)
              o[u] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(*reinterpret_cast<const s16x4*>(w), __builtin_bit_cast(s16x4, u32x2{plane[k][0].x, plane[k][0].y}), o[u], 0, 0, 0);
            else
#pragma unroll
              for (int h = 0; h < PAIRS; ++h)
                o[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const tn_frag*>(w + 8 * h), __builtin_bit_cast(tn_frag, plane[k][h]), o[u], 0, 0, 0);
          }
        } else
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(wc + (((2 * st + u) * CT + ct) * 16 + i) * 16 + 4 * g);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], p[ct][j], o[u], 0, 0, 0);
        }
      }
      const int d = d0 + 32 * st + 8 * g;
      if (!counts) o[0] = o[1] = f32x4{0.f, 0.f, 0.f, 0.f};      // also where the table holds infinity or NaN
      if (in && d < a.D) {
        if constexpr (!WIDE) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (d + e < a.D) {
              if (F32) reinterpret_cast<float*>(a.dx)[t * a.D + d + e] = o[e / 4][e % 4];
              else reinterpret_cast<uint16_t*>(a.dx)[t * a.D + d + e] = to_bf16(o[e / 4][e % 4]);
            }
        } else if (F32) {
          f32x4* to = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.dx) + t * a.D + d);
          to[0] = o[0];
          to[1] = o[1];
        } else
          *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(a.dx) + t * a.D + d) =
              u32x4{pack_bf16(o[0][0], o[0][1]), pack_bf16(o[0][2], o[0][3]), pack_bf16(o[1][0], o[1][1]), pack_bf16(o[1][2], o[1][3])};
      }
    }
    const uint32_t have = (uint32_t)__ballot(counts);    // bit i: row i; what a row without a class holds is not looked at
    constexpr int TOGETHER = (F32 && CT == 6) || (!WIDE && CT * NC == 8) ? 2 : 4;     // (fours spill there)
#pragma unroll TOGETHER
    for (int k = 0; k < 4; ++k) {
      const int row = 4 * k + g;
      const bool has = have >> row & 1;
      const long from = t0 + row < a.T ? t0 + row : a.T - 1;
      float d[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) d[ct] = turned[wave][ct][row][i];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const Few<F32, 4> w = load_few<F32, WIDE, 4>(a.x, from, d0 + 64 * c + 4 * i, a.D);
        f32x4 v;
        if constexpr (F32) v = f32x4{w.v[0], w.v[1], w.v[2], w.v[3]};
        else v = f32x4{__uint_as_float(w.v[0] << 16), __uint_as_float(w.v[0] & 0xffff0000u), __uint_as_float(w.v[1] << 16), __uint_as_float(w.v[1] & 0xffff0000u)};
        if (!has || d0 + 64 * c + 4 * i >= a.D) v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int e = 0; e < 4; ++e) dw[ct][c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(d[ct], v[e], dw[ct][c][e], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

#pragma unroll
  for (int o = 8; o; o >>= 1) { mine.loss += __shfl_xor(mine.loss, o, 64); mine.rows += __shfl_xor(mine.rows, o, 64); }
  if (lane == 0) sums[wave] = mine;
  __syncthreads();
  if (PASS != GRADIENTS && threadIdx.x == 0) {
    RowsPart all = sums[0];
    for (int w = 1; w < 4; ++w) { all.loss += sums[w].loss; all.rows += sums[w].rows; }
    a.parts[blockIdx.x] = all;
  }
  if (PASS == SCORES || !a.dx) return;
  for (int w = 0; w < 4; ++w) {                          // the waves' parts of dW in turn, in the place of W
    if (wave == w) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4* to = reinterpret_cast<f32x4*>(wk + (16 * ct + 4 * g + j) * 64 * NC + 64 * c + 4 * i);
            const f32x4 v{dw[ct][c][0][j], dw[ct][c][1][j], dw[ct][c][2][j], dw[ct][c][3][j]};
            *to = w ? *to + v : v;
          }
    }
    __syncthreads();
  }
  const int width = a.D - d0 < 64 * NC ? a.D - d0 : 64 * NC;
  for (int k = threadIdx.x; k < a.V * width; k += 256) a.part[((long)block * a.V + k / width) * a.D + d0 + k % width] = wk[k / width * 64 * NC + k % width];
}

__global__ __launch_bounds__(256) void count_kernel(const int64_t* __restrict__ target, long T, long V, uint32_t* __restrict__ counts) { count_rows(target, T, V, blockIdx.x, counts); }

// dW from the workgroups' parts: 64 values a workgroup, 16 threads each over the parts; and one more workgroup for the loss
__global__ __launch_bounds__(1024) void few_join_kernel(const float* __restrict__ part, int parts, int n, void* __restrict__ dweight, int bf16, LossArgs l) {
  if (blockIdx.x == 0) {
    sum_loss<1024>(l, nullptr);
    return;
  }
  __shared__ float w[16][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6, k = (blockIdx.x - 1) * 64 + c;
  float s = 0.f;
  if (k < n) {
#pragma unroll 8
    for (int p = q; p < parts; p += 16) s += part[(long)p * n + k];
  }
  w[q][c] = s;
  __syncthreads();
  if (q || k >= n) return;
  for (int p = 1; p < 16; ++p) s += w[p][c];
  if (bf16) reinterpret_cast<uint16_t*>(dweight)[k] = to_bf16(s);
  else reinterpret_cast<float*>(dweight)[k] = s;
}

// ------------------------------------------------------------------------------------------------ host
using Wide = TnTile<256, 256, 2, 4, 2>;
using Mid = TnTile<128, 128, 2, 2, 2>;
using Narrow = TnTile<64, 32, 2, 1, 4>;     // scores of few rows or few tiles: many small workgroups

constexpr long CUS = 256;
// Elements between rows of a buffer of this file's own: whole lines of 64, an odd number of them, so that the rows of a tile do not all start in
// the same few L2 channels (a 4096-wide product took 3 % longer than a 4160-wide one).
long pitch_of(long n) { const long lines = (n + 63) / 64; return (lines | 1) * 64; }

struct Plan {
  bool f32, grad, direct;        // direct: x and W are used where they are
  long T, V, D, Kp, Vp, R, Rp;   // pitches for D and V values; rows of a block, pitch for them
  int blocks, planes, pairs, tile_scores, strips, strip;
  int counters;                  // workgroups that count rows
  int d_planes, d_pairs;         // of d, and products of pairs of planes in the gradients
  size_t inv, counts, rparts, residual, stats, lse, tscore, xp, wp, xt, e, d, dw, part, total, part_bytes;
};

// Which tile for the scores (0: 256 x 256, 1: 128 x 128, 2: 64 x 32): the one with the shortest time by what one step of 64 in k takes a full chip of
// workgroups -- 1.15 us for one a CU, 0.95 for two, 0.48 for three --, what a round of tiles takes besides, and rounds of workgroups.  The smallest are
// for what would leave CUs without a tile (the whole loss in float32, with 128 x 128 and so: 256 x 2000, 1000 classes 220 and 125 us; 4000 x 512, 500
// classes 121 and 113; 1000 x 256, 5000 classes 113 and 129).
int tile_for_scores(long rows, long V, long steps) {
  if (rows <= 32) return 2;      // W streams through once either way: 64 x 32 tiles have it on every CU
  const auto us = [&](long m, long n, long each, double step, double round) {
    return (double)((cdiv(V, m) * (long)cdiv(rows, n) + each * CUS - 1) / (each * CUS)) * ((double)steps * step + round);
  };
  const double t[3] = {us(256, 256, 1, 1.15, 8.0), us(128, 128, 2, 0.95, 6.0), us(64, 32, 3, 0.48, 1.2) + 3.0};
  const int least = t[1] < t[0] ? 1 : 0;
  return t[2] < t[least] ? 2 : least;
}

// Tiles of both gradients, and how many parts of k each is cut to: by the time of one launch that deals out the longer tiles first, a step of 64
// at the rate of a chip that is kept busy and 5 us for a tile's first loads and its results, plus the parts' way through memory (written
// and read once more, at 4 TB/s, and a launch).
struct Shape { int wide, x, w; };
struct Gradients { long D, rows, V, steps_x, steps_w; };
Shape shape_of(const Gradients& g) {
  static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128, 192, 256};
  Shape best{0, 1, 1};
  double least = 1e300;
  for (int wide = 0; wide < 2; ++wide) {
    const long t = wide ? 256 : 128, slots = wide ? CUS : 2 * CUS, nx = cdiv(g.D, t) * (long)cdiv(g.rows, t), nw = cdiv(g.D, t) * (long)cdiv(g.V, t);
    const double step = wide ? 1.65 : 1.36;
    const auto allowed = [&](long s, long n, long steps, long other) { return s == 1 || (s * 8 <= steps && s * g.D * other <= (1L << 28) && n * (s - 1) < 4 * slots); };
    for (const long sx : kSplits) {
      if (!allowed(sx, nx, g.steps_x, g.rows)) break;
      for (const long sw : kSplits) {
        if (!allowed(sw, nw, g.steps_w, g.V)) break;
        double d1 = (double)((g.steps_x + sx - 1) / sx) * step + 5.0, d2 = (double)((g.steps_w + sw - 1) / sw) * step + 5.0;
        long n1 = nx * sx, n2 = nw * sw;
        if (d1 < d2) { const double d = d1; d1 = d2; d2 = d; const long n = n1; n1 = n2; n2 = n; }
        // n1 long tiles leave `busy` of the slots a round behind the others; those take as many short ones as fit meanwhile
        const long rounds = n1 / slots, busy = n1 % slots, fit = (long)(d1 / d2) + 1, ahead = (slots - busy) * fit;
        const long more = n2 <= ahead ? (n2 + slots - busy - 1) / (slots - busy) : fit + (n2 - ahead + slots - 1) / slots;
        const double with_short = (double)rounds * d1 + (double)more * d2, with_long = (double)(rounds + (busy > 0)) * d1;
        double us = with_short > with_long ? with_short : with_long;
        us = 0.7 * us + 0.3 * ((double)n1 * d1 + (double)n2 * d2) / (double)slots;      // CUs that have run out of tiles leave the others their power
        if (sx > 1 || sw > 1) us += 4.0 + ((sx > 1 ? (double)sx * g.rows : 0.0) + (sw > 1 ? (double)sw * g.V : 0.0)) * (double)g.D * 8e-6 / 4.0;
        if (us < least) { least = us; best = Shape{wide, (int)sx, (int)sw}; }
      }
    }
  }
  return best;
}
size_t part_bytes_of(const Shape& s, const Gradients& g) { return ((s.x > 1 ? (size_t)s.x * g.rows : 0) + (s.w > 1 ? (size_t)s.w * g.V : 0)) * g.D * 4; }
Plan plan_of(long T, long V, long D, bool f32, bool grad, bool direct) {
  Plan p{};
  p.f32 = f32; p.grad = grad; p.T = T; p.V = V; p.D = D;
  p.planes = f32 ? 3 : 1;
  p.pairs = f32 ? 6 : 1;
  // d of bfloat16 inputs: one bfloat16 plane.  A row's own entry is most of its d, and what it loses would add as much to dx as dx's own rounding
  // does (0.0024 of the gradient in place of 0.0017), so it is held back in float32 and added in dx's epilogue (4099 x 1000, 50001 classes: 1.484 ms
  // without, 1.498 with it).  In dW it stays, as half a step of bfloat16 at most of each entry, the step to which the result itself is rounded: the row
  // of a class that one row of x has is off by it as a whole, and dW by 0.0020-0.0022 of itself in place of 0.0016-0.0017.  To add it there, the rows of x
  // have to be found by class in every tile, whose first loads then wait for four dependent ones (the same sizes: 1.38 -> 1.47 ms, 1.62 with half of the
  // rows in one class; 4000 x 512, 500 classes 50 -> 61 and 81 us).  For few rows d has two planes and both gradients are exact to their own rounding (8
  // rows, 25840 classes: off by 0.0029 with one plane, 0.0016 with two; 47 and 58 us; 100 rows x 512: 78 and 88 us).
  const bool exact_d = !f32 && T <= 128;
  p.d_planes = f32 ? 3 : exact_d ? 2 : 1;
  p.d_pairs = f32 ? 6 : p.d_planes;
  p.direct = direct && !f32 && D % 64 == 0;
  p.Kp = p.direct ? D : pitch_of(D);
  p.Vp = pitch_of(V);
  const long most = grad ? (1L << (f32 ? 27 : 30)) : (1L << 31);     // (row, class) pairs of a block; without gradients only statistics are held
  p.R = T;
  const long fit = most / V < 1L << 22 ? most / V : 1L << 22;        // 255 rows of x^T stay within 2^32 bytes
  if (T > fit) {            // blocks of one size: whole tiles of rows, or where 256 do not fit, whole steps of 64 of the products over rows
    const long unit = fit >= 256 ? 256 : 64, largest = fit >= unit ? fit / unit * unit : unit, n = (T + largest - 1) / largest;
    p.R = ((T + n - 1) / n + unit - 1) / unit * unit;
    if (p.R > T) p.R = T;
  }
  p.blocks = cdiv(T, p.R);
  p.Rp = pitch_of(p.R);
  p.tile_scores = tile_for_scores(p.R, V, (long)cdiv(D, 64) * p.pairs);
  p.strip = p.tile_scores == 0 ? Wide::WM : p.tile_scores == 1 ? Mid::WM : Narrow::WM;
  p.strips = cdiv(V, p.strip);
  size_t at = 0;
  const auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  p.inv = take(4);
  p.counters = grad ? cdiv(T, COUNTED) : 0;
  p.counts = take((size_t)p.counters * 4);
  p.rparts = take((size_t)(cdiv(T, 32) + 32) * sizeof(RowsPart));
  p.stats = take((size_t)p.strips * p.R * 8);
  p.lse = take((size_t)p.R * 4);
  p.tscore = take((size_t)p.R * 4);
  if (!p.direct) {
    p.xp = take((size_t)p.planes * T * p.Kp * 2);
    p.wp = take((size_t)p.planes * V * p.Kp * 2);
  }
  if (grad) {
    p.residual = take((size_t)p.R * 4);
    p.xt = take((size_t)p.planes * D * p.Rp * 2);
    const size_t held = (size_t)((p.R + 63) / 64 * 64) * p.Vp;
    p.e = take(held * (f32 ? 4 : 2));
    p.d = p.d_planes > 1 ? take(p.d_planes * held * 2) : p.e;
    if (p.blocks > 1 && !f32) p.dw = take((size_t)V * D * 4);
    const Gradients g{D, p.R, V, (long)cdiv(V, 64) * p.d_pairs, (long)cdiv(p.R, 64) * p.d_pairs};
    p.part_bytes = part_bytes_of(shape_of(g), g);
    p.part = take(p.part_bytes);
  }
  p.total = at;
  return p;
}

template <class T, bool F32>
int launch_scores(TnArgs g, const ScoreOut& o, hipStream_t st) {
  DPPM_TRY(lds_limit(reinterpret_cast<const void*>(scores_kernel<T, F32>), T::LDS, "dppm_loss_ce"));
  g.tiles_m = cdiv(g.M, T::BM);
  g.tiles_n = cdiv(g.N, T::BN);
  hipLaunchKernelGGL((scores_kernel<T, F32>), dim3(g.tiles_m * g.tiles_n), dim3(T::NT), T::LDS, st, g, o);
  return DPPM_OK;
}

template <class T>
void launch_gradients(GradJob x, GradJob w, hipStream_t st, int& rc) {
  rc = lds_limit(reinterpret_cast<const void*>(grad_kernel<T>), T::LDS, "dppm_loss_ce");
  if (rc != DPPM_OK) return;
  const auto tiles = [](GradJob& j) {
    j.g.tiles_m = cdiv(j.g.M, T::BM);
    j.g.tiles_n = cdiv(j.g.N, T::BN);
    return j.g.tiles_m * j.g.tiles_n * j.g.splits;
  };
  const int nx = tiles(x), nw = tiles(w);
  const bool w_first = (long)w.g.ksteps * w.g.pairs * x.g.splits > (long)x.g.ksteps * x.g.pairs * w.g.splits;
  hipLaunchKernelGGL((grad_kernel<T>), dim3(nx + nw), dim3(T::NT), T::LDS, st, x, w, w_first ? nw : nx, (int)w_first);
}

GradJob grad_job(const TnArgs& g, void* c, bool c_bf16, const float* scale) {
  GradJob j{};
  j.g = g;
  j.o.c = c; j.o.ldc = g.M; j.o.c_bf16 = c_bf16; j.o.scale = scale;
  j.o.past = (size_t)g.M * g.N * (c_bf16 ? 2 : 4) > CACHED;
  j.o.wide = g.M % 8 == 0 && (uintptr_t)c % 16 == 0;
  return j;
}

// dx[n][m] = sum_k A[m][k] B[n][k] over the classes, and dW (+= add) over the rows
int gradients(GradJob x, GradJob w, float* part, size_t part_bytes, hipStream_t st) {
  const Gradients g{x.g.M, x.g.N, w.g.N, (long)x.g.ksteps * x.g.pairs, (long)w.g.ksteps * w.g.pairs};
  Shape shape = shape_of(g);
  if (part_bytes_of(shape, g) > part_bytes) shape.x = shape.w = 1;      // a last, smaller block of rows
  const auto cut = [&](GradJob& j, int splits) {
    PartsJob p{part, (long)j.g.M * j.g.N, splits, j.o.add, j.o.c, j.o.c_bf16};
    j.g.splits = splits;
    if (splits == 1) { p.n = 0; return p; }
    j.o.part = part; j.o.part_stride = p.n; j.o.add = nullptr;
    part += splits * p.n;
    return p;
  };
  const PartsJob px = cut(x, shape.x), pw = cut(w, shape.w);
  int rc;
  if (shape.wide) launch_gradients<Wide>(x, w, st, rc);
  else launch_gradients<Mid>(x, w, st, rc);
  DPPM_TRY(rc);
  const auto blocks = [](const PartsJob& p) { const long b = (p.n + 255) / 256; return (int)(b < 8192 ? b : 8192); };
  const int bx = blocks(px), bw = blocks(pw);
  if (bx + bw) hipLaunchKernelGGL(parts_kernel, dim3(bx + bw), dim3(256), 0, st, px, pw, bx);
  return DPPM_OK;
}

// few_kernel: the rule on sizes, and its workspace.  Losses and gradients in one pass and by the products in tiles, which pad the classes to 128 and
// hold x^T, scores and d in memory, bfloat16 / float32: 2^20 rows x 64, 5 classes 87 / 137 us and 443 / 1289 (60 / 118 at a copy's rate); at its largest
// sizes, 2^16 x 512, 16 classes 57 / 90 and 98 / 350, x 128, 64 classes 42 / 67 and 58 / 113, x 64, 128 classes 61 / 71 and 65 / 117 (losses alone 20 / 29
// and 17 / 40); 1000 x 64, 100 classes 20 / 24 and 33 / 47.  Rows that are not aligned are read value by value: 2^20 x 63, 5 classes 217 / 313 and 714 / 1463.
struct FewPlan { bool fits, two; int ct, nc, grid, slices, blocks, counters, lds; size_t counts, parts, d, part, total; };
FewPlan few_plan(long T, long V, long D, bool f32, bool grad, bool wide) {
  FewPlan f{};
  f.ct = V <= 16 ? 1 : V <= 32 ? 2 : V <= 64 ? 4 : V <= 96 ? 6 : 8;
  f.nc = D <= 64 ? 1 : D <= 128 ? 2 : D <= 256 ? 4 : 8;
  if (V > FEW_CLASSES) return f;
  const long groups = (T + 63) / 64;
  if (f.ct * f.nc * 64 <= FEW_VALUES && D <= FEW_VALUES) {
    const long most = CUS * (f.ct * f.nc <= 2 ? 4 : 2);
    f.grid = f.blocks = (int)(groups < most ? groups : most);
    f.slices = 1;
  } else {
    // In two passes, with all of W in LDS in one order and d of T rows in memory; in tiles and so, bfloat16 / float32: 2^16 x 1024, 5 classes 193 / 663 and
    // 99 / 209 us; 8192 x 256, 40 classes 34 / 59 and 29 / 35; 1000 x 1024, 5 classes 34 / 73 and 27 / 34.  bfloat16 with more than 64 classes (8192 x
    // 256, 100 classes 38 and 44) or unaligned rows (1000 x 777, 20 classes 39 and 54), and its losses alone, stay in tiles.
    f.lds = f.ct * cdiv(D, 128) * (f32 ? 8192 : 4096);
    if (f.lds > (128 << 10) || T * f.ct > (1L << 24) || !(f32 || (grad && wide && f.ct <= 4))) return f;
    f.two = true;
    f.nc = f.ct == 6 ? 1 : 8 / f.ct;
    f.slices = cdiv(D, 64 * f.nc);
    const long one = CUS * (f.lds > (72 << 10) ? 1 : 2), two = 2 * CUS / f.slices;
    f.grid = (int)(groups < one ? groups : one);
    f.blocks = (int)(groups < two ? groups : two < 1 ? 1 : two);
  }
  f.fits = true;
  f.counters = grad && T > COUNTED ? cdiv(T, COUNTED) : 0;
  f.parts = ((size_t)f.counters * 4 + 255) / 256 * 256;
  f.d = f.parts + ((size_t)f.grid * sizeof(RowsPart) + 255) / 256 * 256;
  f.part = f.d + (grad && f.two ? (size_t)T * f.ct * 64 : 0);
  f.total = f.part + (grad ? (size_t)f.blocks * V * D * 4 : 0);
  return f;
}
template <bool F32, bool WIDE, int CT, int NC, FewPass PASS>
int launch_few(const FewArgs& a, int grid, int lds, hipStream_t st) {
  DPPM_TRY(lds_limit(reinterpret_cast<const void*>(few_kernel<F32, WIDE, CT, NC, PASS>), lds, "dppm_loss_ce"));
  hipLaunchKernelGGL((few_kernel<F32, WIDE, CT, NC, PASS>), dim3(grid), dim3(256), lds, st, a);
  return DPPM_OK;
}
template <bool F32, bool WIDE, int CT, int NC>
int one_pass(const FewPlan& f, const FewArgs& a, hipStream_t st) { return launch_few<F32, WIDE, CT, NC, ALL>(a, f.grid, NC * CT * (F32 ? 8192 : 4096), st); }
template <bool F32, bool WIDE, int CT, int NC>
int two_passes(const FewPlan& f, const FewArgs& a, hipStream_t st) {
  DPPM_TRY((launch_few<F32, WIDE, CT, NC, SCORES>(a, f.grid, f.lds, st)));
  return a.dx ? launch_few<F32, WIDE, CT, NC, GRADIENTS>(a, f.blocks * f.slices, NC * CT * 4096, st) : DPPM_OK;
}
template <bool F32, bool WIDE>
int few_classes(const FewPlan& f, FewArgs a, bool denominator, float* loss, void* dweight, char* ws, hipStream_t st) {
  a.counts = reinterpret_cast<uint32_t*>(ws + f.counts);
  a.parts = reinterpret_cast<RowsPart*>(ws + f.parts);
  a.part = reinterpret_cast<float*>(ws + f.part);
  a.d = reinterpret_cast<float*>(ws + f.d);
  a.slices = f.slices;
  a.counters = denominator ? 0 : f.counters;
  if (a.counters) hipLaunchKernelGGL(count_kernel, dim3(a.counters), dim3(256), 0, st, a.target, a.T, (long)a.V, reinterpret_cast<uint32_t*>(ws + f.counts));
  if (f.two) {
    if constexpr (F32 || WIDE) {
      if (f.ct == 1) DPPM_TRY((two_passes<F32, WIDE, 1, 8>(f, a, st)));
      else if (f.ct == 2) DPPM_TRY((two_passes<F32, WIDE, 2, 4>(f, a, st)));
      else if (f.ct == 4) DPPM_TRY((two_passes<F32, WIDE, 4, 2>(f, a, st)));
      if constexpr (F32) {
        if (f.ct == 6) DPPM_TRY((two_passes<F32, WIDE, 6, 1>(f, a, st)));
        else if (f.ct == 8) DPPM_TRY((two_passes<F32, WIDE, 8, 1>(f, a, st)));
      }
    }
  } else if (f.ct == 1) {
    if (f.nc == 1) DPPM_TRY((one_pass<F32, WIDE, 1, 1>(f, a, st)));
    else if (f.nc == 2) DPPM_TRY((one_pass<F32, WIDE, 1, 2>(f, a, st)));
    else if (f.nc == 4) DPPM_TRY((one_pass<F32, WIDE, 1, 4>(f, a, st)));
    else DPPM_TRY((one_pass<F32, WIDE, 1, 8>(f, a, st)));
  } else if (f.ct == 2) {
    if (f.nc == 1) DPPM_TRY((one_pass<F32, WIDE, 2, 1>(f, a, st)));
    else if (f.nc == 2) DPPM_TRY((one_pass<F32, WIDE, 2, 2>(f, a, st)));
    else DPPM_TRY((one_pass<F32, WIDE, 2, 4>(f, a, st)));
  } else if (f.ct == 4) {
    if (f.nc == 1) DPPM_TRY((one_pass<F32, WIDE, 4, 1>(f, a, st)));
    else DPPM_TRY((one_pass<F32, WIDE, 4, 2>(f, a, st)));
  } else if (f.ct == 6)
    DPPM_TRY((one_pass<F32, WIDE, 6, 1>(f, a, st)));
  else
    DPPM_TRY((one_pass<F32, WIDE, 8, 1>(f, a, st)));
  const int n = a.dx ? a.V * a.D : 0;
  hipLaunchKernelGGL(few_join_kernel, dim3(1 + cdiv(n, 64)), dim3(1024), 0, st, a.part, f.blocks, n, dweight, (int)!F32, LossArgs{a.parts, f.grid, a.denom, loss});
  return DPPM_OK;
}

// -> workgroups for it
int lay_out(LayOut& a, bool f32, const void* src, long rows, long cols, uint16_t* as_is, long pitch, uint16_t* turned, long pitch_t, const int64_t* target, long V) {
  const long r = turned && pitch_t > rows ? pitch_t : rows, c = as_is ? pitch : cols;
  a = LayOut{src, (int)rows, (int)cols, as_is, pitch, rows * pitch, turned, pitch_t, cols * pitch_t, target, V, cdiv(c, 64),
             (uintptr_t)src % 16 == 0 && cols % (f32 ? 4 : 8) == 0};
  return a.across * cdiv(r, 64);
}

bool sizes_ok(int64_t T, int64_t V, int64_t D) { return T >= 0 && V >= 1 && D >= 1 && T < (1L << 30) && V <= (1L << 23) && D <= (1L << 16); }   // 255 rows of any operand lie within 2^32 bytes

}  // namespace
}  // namespace dppm

using namespace dppm;

extern "C" size_t dppm_loss_ce_workspace_bytes(int64_t T, int64_t V, int64_t D, int bf16, int want_grad) {
  if (!sizes_ok(T, V, D) || T == 0) return 0;
  const size_t tiles = plan_of(T, V, D, !bf16, want_grad, false).total, few = few_plan(T, V, D, !bf16, want_grad, true).total;
  return tiles > few ? tiles : few;      // the largest of the layouts, so that the size does not depend on addresses
}

extern "C" int dppm_loss_ce_fwd_bwd(const void* x, const void* weight, int bf16, const int64_t* target, const float* row_weight, double denom, int64_t T,
                                    int64_t V, int64_t D, float* loss_out, float* row_loss, void* dx, void* dweight, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  DPPM_REQUIRE(sizes_ok(T, V, D), "dppm_loss_ce_fwd_bwd: T=%ld V=%ld D=%ld", (long)T, (long)V, (long)D);
  DPPM_REQUIRE(denom == 0 || (denom >= 1e-37 && denom <= 1e37), "dppm_loss_ce_fwd_bwd: denom=%g", denom);
  DPPM_REQUIRE(T >= 1, "dppm_loss_ce_fwd_bwd: no rows");
  DPPM_REQUIRE(x && weight && target && loss_out && row_loss && workspace, "dppm_loss_ce_fwd_bwd: null pointer");
  DPPM_REQUIRE((dx == nullptr) == (dweight == nullptr), "dppm_loss_ce_fwd_bwd: dx and dweight come together");
  DPPM_REQUIRE((uintptr_t)workspace % 16 == 0, "dppm_loss_ce_fwd_bwd: the workspace must be 16-byte aligned");
  const bool grad = dx != nullptr, aligned = ((uintptr_t)x | (uintptr_t)weight) % 16 == 0;
  const bool wide = D % 8 == 0 && aligned && (uintptr_t)dx % 16 == 0;
  const FewPlan few = few_plan(T, V, D, !bf16, grad, wide);
  if (few.fits) {
    DPPM_REQUIRE(workspace_bytes >= few.total, "dppm_loss_ce_fwd_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, few.total);
    const FewArgs a{x, weight, target, row_weight, nullptr, 0, (long)T, (int)V, (int)D, (float)denom, row_loss, dx, nullptr, nullptr, nullptr, 1};
    const auto run = bf16 ? (wide ? few_classes<false, true> : few_classes<false, false>) : (wide ? few_classes<true, true> : few_classes<true, false>);
    DPPM_TRY(run(few, a, denom > 0, loss_out, dweight, reinterpret_cast<char*>(workspace), as_stream(stream)));
    return check_launch("dppm_loss_ce_fwd_bwd");
  }
  const Plan p = plan_of(T, V, D, !bf16, grad, aligned);
  DPPM_REQUIRE(workspace_bytes >= p.total, "dppm_loss_ce_fwd_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, p.total);
  const hipStream_t st = as_stream(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  const auto h = [&](size_t at) { return reinterpret_cast<uint16_t*>(ws + at); };
  const auto f = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
  float2* stats = reinterpret_cast<float2*>(ws + p.stats);
  const uint16_t *xp = reinterpret_cast<const uint16_t*>(x), *wp = reinterpret_cast<const uint16_t*>(weight);
  const size_t es = bf16 ? 2 : 4;
  RowsPart* const parts = reinterpret_cast<RowsPart*>(ws + p.rparts);
  uint32_t* const counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  int sums = 0;      // parts written so far
  const auto prepare = [&](const LayOut& a, int first, const LayOut& b, int second, int counters) {
    const int grid = first + second + counters;
    if (grid == 0) return;
    if (p.f32) hipLaunchKernelGGL((prepare_kernel<true>), dim3(grid), dim3(256), 0, st, a, first, b, second, target, (long)T, (long)V, counts);
    else hipLaunchKernelGGL((prepare_kernel<false>), dim3(grid), dim3(256), 0, st, a, first, b, second, target, (long)T, (long)V, counts);
  };
  {
    // a single block's transposed x is made here too; rows of x without a class are zeros in both, which changes nothing that counts
    LayOut w{}, xs{};
    int first = 0, second = 0;
    const bool turn_x = grad && p.blocks == 1;
    if (!p.direct) first = lay_out(w, p.f32, weight, V, D, h(p.wp), p.Kp, nullptr, 0, nullptr, 0);
    if (!p.direct || turn_x) second = lay_out(xs, p.f32, x, T, D, p.direct ? nullptr : h(p.xp), p.Kp, turn_x ? h(p.xt) : nullptr, p.Rp, target, V);
    prepare(w, first, xs, second, p.counters);
    if (!p.direct) { xp = h(p.xp); wp = h(p.wp); }
  }
  for (int b = 0; b < p.blocks; ++b) {
    const long t0 = b * p.R, rows = T - t0 < p.R ? T - t0 : p.R, Rp = pitch_of(rows);
    TnArgs g{};
    g.A = wp; g.lda = p.Kp; g.plane_a = V * p.Kp; g.M = (int)V;
    g.B = xp + t0 * p.Kp; g.ldb = p.Kp; g.plane_b = T * p.Kp; g.N = (int)rows;
    g.K = (int)D; g.ksteps = cdiv(D, 64); g.pairs = p.pairs; g.splits = 1;
    ScoreOut o{};
    o.stats = stats; o.target_score = f(p.tscore); o.target = target + t0; o.e = grad ? ws + p.e : nullptr; o.pitch = p.Vp; o.V = (int)V;
    o.past = (size_t)rows * p.Vp * (p.f32 ? 4 : 2) > CACHED;
    if (p.tile_scores == 0) DPPM_TRY(p.f32 ? (launch_scores<Wide, true>(g, o, st)) : (launch_scores<Wide, false>(g, o, st)));
    else if (p.tile_scores == 1) DPPM_TRY(p.f32 ? (launch_scores<Mid, true>(g, o, st)) : (launch_scores<Mid, false>(g, o, st)));
    else DPPM_TRY(p.f32 ? (launch_scores<Narrow, true>(g, o, st)) : (launch_scores<Narrow, false>(g, o, st)));
    const RowsArgs r{stats, p.strips, (int)rows, target + t0, (long)V, f(p.tscore), row_weight ? row_weight + t0 : nullptr, f(p.lse), row_loss + t0, parts + sums};
    if (!grad && T <= 8) {
      hipLaunchKernelGGL(rows_and_loss_kernel, dim3(1), dim3(1024), 0, st, r, (float)denom, loss_out);
      break;
    }
    // a thread's share of the strips is what takes the time: with few rows, more threads a row
    const int by = T <= 64 ? 2 : 32, n = cdiv(rows, by);
    const bool join = grad && b == 0;
    if (by == 2) hipLaunchKernelGGL((rows_kernel<2>), dim3(n + join), dim3(256), 0, st, r, join ? counts : nullptr, p.counters, (float)denom, f(p.inv));
    else hipLaunchKernelGGL((rows_kernel<32>), dim3(n + join), dim3(256), 0, st, r, join ? counts : nullptr, p.counters, (float)denom, f(p.inv));
    sums += n;
    if (!grad) continue;
    const int whole = cdiv(rows, 64) * 64;
    TurnArgs a{};
    a.e = ws + p.e; a.pitch = p.Vp; a.stats = stats; a.lse = f(p.lse); a.target_score = f(p.tscore); a.target = target + t0;
    a.row_weight = row_weight ? row_weight + t0 : nullptr; a.inv = f(p.inv);
    a.residual = f(p.residual); a.d = h(p.d); a.plane = whole * p.Vp; a.rows = (int)rows; a.V = (int)V; a.strip = p.strip; a.past = (size_t)p.d_planes * a.plane * 2 > CACHED;
    const bool last = b == p.blocks - 1;
    const LossArgs sum{parts, sums, (float)denom, last ? loss_out : nullptr};
    const int lanes = p.Vp <= 64 && p.d_planes != 2 ? 8 : 64;
    a.whole = whole;
    a.across = cdiv(p.Vp, 8 * lanes);
    const dim3 grid((unsigned)((long)a.across * cdiv(whole, 1024 / lanes) + 1));      // (a second dimension of a grid ends at 65535)
    if (p.f32) {
      if (lanes == 8) hipLaunchKernelGGL((turn_kernel<true, 3, 8>), grid, dim3(256), 0, st, a, sum);
      else hipLaunchKernelGGL((turn_kernel<true, 3, 64>), grid, dim3(256), 0, st, a, sum);
    } else if (p.d_planes == 2) hipLaunchKernelGGL((turn_kernel<false, 2, 64>), grid, dim3(256), 0, st, a, sum);
    else if (lanes == 8) hipLaunchKernelGGL((turn_kernel<false, 1, 8>), grid, dim3(256), 0, st, a, sum);
    else hipLaunchKernelGGL((turn_kernel<false, 1, 64>), grid, dim3(256), 0, st, a, sum);
    if (p.blocks > 1) {
      LayOut xs{};
      const int n = lay_out(xs, p.f32, reinterpret_cast<const char*>(x) + t0 * D * es, rows, D, nullptr, 0, h(p.xt), Rp, target + t0, V);
      prepare(xs, n, xs, 0, 0);
    }
    TnArgs gx{};       // dx[t][d] = sum_v d[t][v] W[v][d]
    gx.A = wp; gx.lda = p.Kp; gx.plane_a = V * p.Kp; gx.M = (int)D;
    gx.B = a.d; gx.ldb = p.Vp; gx.plane_b = a.plane; gx.N = (int)rows;
    gx.K = (int)V; gx.ksteps = cdiv(V, 64); gx.pairs = p.d_pairs;
    TnArgs gw{};       // dW[v][d] = sum_t d[t][v] x^T[d][t]
    gw.A = h(p.xt); gw.lda = Rp; gw.plane_a = D * Rp; gw.M = (int)D;
    gw.B = a.d; gw.ldb = p.Vp; gw.plane_b = a.plane; gw.N = (int)V;
    gw.K = whole; gw.ksteps = cdiv(rows, 64); gw.pairs = p.d_pairs;      // d has zeros to whole steps
    float* total = p.blocks == 1 ? nullptr : (p.f32 ? reinterpret_cast<float*>(dweight) : f(p.dw));
    GradJob jx = grad_job(gx, reinterpret_cast<char*>(dx) + t0 * D * es, bf16, f(p.inv));
    jx.o.target = target + t0;
    if (p.d_planes == 1) jx.o.residual = f(p.residual);
    GradJob jw = grad_job(gw, last || p.f32 ? dweight : (void*)total, bf16 && last, f(p.inv));
    jw.o.add = b == 0 ? nullptr : total;
    DPPM_TRY(gradients(jx, jw, f(p.part), p.part_bytes, st));
  }
  if (!grad && T > 8) hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, LossArgs{parts, sums, (float)denom, loss_out});
  return check_launch("dppm_loss_ce_fwd_bwd");
}

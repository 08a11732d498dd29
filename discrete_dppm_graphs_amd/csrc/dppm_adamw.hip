// AdamW over many tensors in one launch, with the moments in float32 or in 8 bits, and the gradient's norm clipped in the same call.
//
//   g' = g * grad_scale * min(1, max_norm / (|g * grad_scale| + 1e-6))          |.|: over all tensors together, summed in float64
//   m' = m + (1 - beta1) (g' - m)          v' = beta2 v + (1 - beta2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - beta1^t) * m' / (sqrt(v') / sqrt(1 - beta2^t) + eps)
//
// HBM-bound: with float32 moments 28 bytes a value (float32 gradient), with 8-bit moments and a bfloat16 gradient and copy 16.
// A table of tensors and a table of chunks (both on the device, laid out once by the caller) make every workgroup's work one lookup
// away, whatever the number of tensors: launches do not grow with it.
//
// 8-bit moments.  Held are m and r = sqrt(v) as e4m3 (OCP: 3 mantissa bits, 2^-9 .. 448) with one float32 scale per 256 consecutive
// values of a tensor, scale = (largest magnitude) / 448.  The root and not v itself: e4m3 spans 2^17.8, so that r spans the range of
// gradients within a block and v its square.  The rounding is stochastic: beta2 = 0.999 moves v by 1e-3 of itself in a step while half
// a step of e4m3 is up to 6e-2, so that rounding to nearest would never let a second moment fall.  Rounded up with the probability of
// the dropped part, r follows the exact recursion in the mean.  The update itself uses m' and v' before they are rounded.
// Random bits: Philox4x32-10, key = seed, counter = (group, tensor, group >> 32, step), group = index in the tensor / 4; word k of the
// four belongs to value 4 group + k, its high 16 bits to m and its low 16 bits to r.
#include <cmath>
#include "dppm_common.h"
#include "dppm_philox.h"

namespace dppm {
namespace {

constexpr int BLK = 256;           // values that share a scale = one quad of values on each lane of a wave
constexpr int CHUNK = 4096;        // values of one workgroup: 256 threads x 4 quads
constexpr int NORM_GRID = 2048;    // partial sums of the gradient's norm: as many workgroups as the chip holds

struct StepArgs {
  float one_minus_b1, b2, one_minus_b2, eps, step_size, bc2_rsqrt, gscale;
  double lr;
  uint32_t step;
  uint2 key;
};

struct NormOut { float mult; int ok; };   // what the step reads: the gradient's factor, and whether the norm is finite

// The table's pointers are global memory: said so, the loads and stores are global ones and not flat ones, which also count as LDS accesses.
template <class T> using glb = __attribute__((address_space(1))) T*;
template <class T> __device__ __forceinline__ glb<T> global(T* p) { return (glb<T>)p; }
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_to_f32(uint32_t b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ uint32_t f32_to_bf16x2(float lo, float hi) {   // round to nearest even (one instruction on gfx950)
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}

// the value of an e4m3 code: its 7 magnitude bits put on float32's exponent and mantissa are the value times 2^-120, denormals included
__device__ __forceinline__ float e4m3_value(uint32_t code) { return __uint_as_float(((code & 0x80u) << 24) | ((code & 0x7fu) << 20)) * 0x1p120f; }

// codes of |x| * inv (<= 448 up to a rounding), rounded up with probability (dropped part) by 16 random bits each.  Above 2^-6 the
// random bits are added to the 20 mantissa bits that go; below, the grid is the constant 2^-9: few values are (under 2^-15 of their
// block's largest), so that a wave without one skips that form.
template <bool SIGNED>
__device__ __forceinline__ uint32_t e4m3_codes(const float (&x)[4], float inv, const uint32_t (&r16)[4]) {
  float y[4];
  uint32_t code[4], out = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    y[k] = fminf(fabsf(x[k]) * inv, 448.f);
    code[k] = ((__float_as_uint(y[k]) + (r16[k] << 4)) >> 20) - 960u;
  }
  if (__any(fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) < 0x1p-6f)) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (y[k] < 0x1p-6f) code[k] = (uint32_t)(y[k] * 512.f + (float)r16[k] * 0x1p-16f);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    code[k] = code[k] < 126u ? code[k] : 126u;
    if (SIGNED) code[k] |= (__float_as_uint(x[k]) >> 24) & 0x80u;
    out |= code[k] << (8 * k);
  }
  return out;
}

// largest of non-negative floats over a wave, on their bit patterns: a NaN is larger than infinity there and is kept, so that a block with
// a NaN in it gets a NaN for its scale and reads back as NaN throughout, instead of as 448 in one place
__device__ __forceinline__ float wave_max(uint32_t v) {
#define DPPM_MAX_STEP(ctrl)                                                                    \
  {                                                                                            \
    const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true); \
    v = v > w ? v : w;                                                                         \
  }
  DPPM_MAX_STEP(0x111)   // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has the row's maximum (a lane without a source reads 0)
  DPPM_MAX_STEP(0x112)
  DPPM_MAX_STEP(0x114)
  DPPM_MAX_STEP(0x118)
  DPPM_MAX_STEP(0x142)   // row_bcast:15, row_bcast:31: lane 63 has the wave's
  DPPM_MAX_STEP(0x143)
#undef DPPM_MAX_STEP
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)v, 63));
}
__device__ __forceinline__ uint32_t magnitude_max(uint32_t v, float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return v > b ? v : b;
}

// v_sqrt_f32 takes denormal operands as zero, which with eps = 0 would divide by it
__device__ __forceinline__ float fast_root(float v) {
  const bool tiny = v < 0x1p-126f;
  return __builtin_amdgcn_sqrtf(tiny ? v * 0x1p64f : v) * (tiny ? 0x1p-32f : 1.f);
}

// four values from `at` on; FULL: all of them lie before the tensor's end, n values long
template <bool BF, bool FULL>
__device__ __forceinline__ void load4(const void* src, long at, long n, float (&out)[4]) {
  if (BF) {
    const glb<const uint16_t> q = (glb<const uint16_t>)src + at;
    if (FULL || at + 4 <= n) {
      const u32x2 w = *(glb<const u32x2>)q;
      out[0] = bf16_to_f32(w.x & 0xffffu); out[1] = __uint_as_float(w.x & 0xffff0000u);
      out[2] = bf16_to_f32(w.y & 0xffffu); out[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = at + k < n ? bf16_to_f32(q[k]) : 0.f;
    }
  } else {
    const glb<const float> q = (glb<const float>)src + at;
    if (FULL || at + 4 <= n) {
      const f32x4 w = *(glb<const f32x4>)q;
      out[0] = w.x; out[1] = w.y; out[2] = w.z; out[3] = w.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = at + k < n ? q[k] : 0.f;
    }
  }
}
template <bool FULL>
__device__ __forceinline__ void store4(void* dst, long at, long n, const float (&v)[4]) {
  const glb<float> q = (glb<float>)dst + at;
  if (FULL || at + 4 <= n) *(glb<f32x4>)q = f32x4{v[0], v[1], v[2], v[3]};
  else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k < n) q[k] = v[k];
  }
}

// sum of squares of all gradients: every workgroup walks chunks at a fixed stride, so that the partial sums, and their sum below, are
// the same from call to call
template <bool GBF>
__global__ __launch_bounds__(256) void grad_sq_kernel(const dppm_tensor_entry* __restrict__ tab, const int2* __restrict__ chunks, int n_chunks,
                                                      double* __restrict__ part) {
  double s = 0.0;
  // two chunks at a time: a chunk's loads wait for its table entry, which waits for its pair
  for (int c = blockIdx.x; c < n_chunks; c += 2 * gridDim.x) {
    float q[2][4][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool in = c + j * (int)gridDim.x < n_chunks;
      const int2 ch = chunks[in ? c + j * (int)gridDim.x : c];
      const void* g = tab[ch.x].grad;
      const long n = in ? tab[ch.x].numel : 0, base = (long)ch.y * CHUNK;
      if (base + CHUNK <= n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load4<GBF, true>(g, base + (i * 256 + threadIdx.x) * 4, n, q[j][i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) load4<GBF, false>(g, base + (i * 256 + threadIdx.x) * 4, n, q[j][i]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s += (double)q[j][i][k] * (double)q[j][i][k];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
  __shared__ double w[4];
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}

// The partial sums of all workgroups, by 256 threads in a fixed order: the norm, and what the step reads.  All threads get the result.
__device__ __forceinline__ NormOut clip_of(const double* part, int n, double gscale, double max_norm, float* norm_out) {
  __shared__ double w[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((w[0] + w[1]) + (w[2] + w[3])) * fabs(gscale);
  const double coef = max_norm / (norm + 1e-6);
  if (norm_out && threadIdx.x == 0) *norm_out = (float)norm;
  // not ok where the caller reads infinity (a float32) or NaN: the step leaves everything as it was
  return NormOut{(float)(gscale * (coef < 1.0 ? coef : 1.0)), (float)norm <= 3.402823466e38f};
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* __restrict__ part, int n, double gscale, double max_norm, float* __restrict__ norm_out,
                                                        NormOut* __restrict__ out) {
  const NormOut o = clip_of(part, n, gscale, max_norm, norm_out);
  if (threadIdx.x == 0) *out = o;
}

template <bool GBF, int BITS, bool FULL>
__device__ __forceinline__ void adamw_chunk(const dppm_tensor_entry& e, long base, uint32_t tensor, float mult, const StepArgs& a) {
  const long n = e.numel;
  const float decay = (float)(1.0 - a.lr * e.weight_decay);
  float p[4][4], g[4][4], m[4][4], v[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long at = base + (i * 256 + threadIdx.x) * 4;
    load4<GBF, FULL>(e.grad, at, n, g[i]);
    load4<false, FULL>(e.param, at, n, p[i]);
    if (BITS == 32) {
      load4<false, FULL>(e.exp_avg, at, n, m[i]);
      load4<false, FULL>(e.exp_avg_sq, at, n, v[i]);
    } else {   // 8-bit moments are padded to whole blocks, so that whole words are read and written
      uint32_t cm = 0, cr = 0;
      float sm = 0.f, sr = 0.f;
      if (FULL || at < n) {
        cm = ((glb<const uint32_t>)e.exp_avg)[at >> 2];
        cr = ((glb<const uint32_t>)e.exp_avg_sq)[at >> 2];
        sm = global(e.exp_avg_scale)[at / BLK];
        sr = global(e.exp_avg_sq_scale)[at / BLK];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[i][k] = e4m3_value(cm >> (8 * k)) * sm;
        const float r = e4m3_value(cr >> (8 * k)) * sr;
        v[i][k] = r * r;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long at = base + (i * 256 + threadIdx.x) * 4;
    float root[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gg = g[i][k] * mult;
      m[i][k] = m[i][k] + (gg - m[i][k]) * a.one_minus_b1;
      v[i][k] = v[i][k] * a.b2 + a.one_minus_b2 * gg * gg;
      // the hardware's root and reciprocal are off by one unit in the last place: enough for the update, which is small against p.  A root
      // that is stored is rounded correctly.  (eps = 0: v' is 0 or at least 2^-149, so that the denominator is 0 or far from the denormals.)
      root[k] = BITS == 8 ? sqrtf(v[i][k]) : fast_root(v[i][k]);
      p[i][k] = p[i][k] * decay - a.step_size * (m[i][k] * __builtin_amdgcn_rcpf(root[k] * a.bc2_rsqrt + a.eps));
    }
    if (BITS == 8) {
      // values behind the tensor's end count as zero: in the block's maximum and in the padding that is written
      uint32_t um = 0, ur = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!FULL && at + k >= n) { m[i][k] = 0.f; root[k] = 0.f; }
        um = magnitude_max(um, m[i][k]);
        ur = magnitude_max(ur, root[k]);
      }
      const float tm = wave_max(um), tr = wave_max(ur);
      if (FULL || at < n) {
        // a block whose largest value is under 1e-30 is held as zero: its reciprocal would overflow.  (The comparison is false for NaN.)
        const float im = tm <= 1e-30f ? 0.f : 1.f / tm * 448.f, ir = tr <= 1e-30f ? 0.f : 1.f / tr * 448.f;
        const uint64_t group = (uint64_t)at >> 2;
        const uint4 rnd = philox4x32_10_mad(make_uint4((uint32_t)group, tensor, (uint32_t)(group >> 32), a.step), a.key);
        const uint32_t rm[4] = {rnd.x >> 16, rnd.y >> 16, rnd.z >> 16, rnd.w >> 16};
        const uint32_t rr[4] = {rnd.x & 0xffffu, rnd.y & 0xffffu, rnd.z & 0xffffu, rnd.w & 0xffffu};
        ((glb<uint32_t>)e.exp_avg)[at >> 2] = e4m3_codes<true>(m[i], im, rm);
        ((glb<uint32_t>)e.exp_avg_sq)[at >> 2] = e4m3_codes<false>(root, ir, rr);
        if ((threadIdx.x & 63) == 0) {
          global(e.exp_avg_scale)[at / BLK] = tm <= 1e-30f ? 0.f : tm * (1.f / 448.f);
          global(e.exp_avg_sq_scale)[at / BLK] = tr <= 1e-30f ? 0.f : tr * (1.f / 448.f);
        }
      }
    }
    store4<FULL>(e.param, at, n, p[i]);
    if (BITS == 32) {
      store4<FULL>(e.exp_avg, at, n, m[i]);
      store4<FULL>(e.exp_avg_sq, at, n, v[i]);
    }
    if (e.copy) {
      const glb<uint16_t> c = global(e.copy) + at;
      const uint32_t lo = f32_to_bf16x2(p[i][0], p[i][1]), hi = f32_to_bf16x2(p[i][2], p[i][3]);
      if (FULL || at + 4 <= n) *(glb<u32x2>)c = u32x2{lo, hi};
      else {
        if (at < n) c[0] = (uint16_t)lo;
        if (at + 1 < n) c[1] = (uint16_t)(lo >> 16);
        if (at + 2 < n) c[2] = (uint16_t)hi;
      }
    }
  }
}

// clip: what grad_norm_kernel left; or null, and with parts > 0 every workgroup sums the few partial sums itself, which spares the launch.  Clipped
// float32 steps with the launch and without it, in us: 512 chunks 14.0 / 11.4, 600 17.8 / 16.0, 1024 25.4 / 23.1, 2048 47.0 / 43.7, 4096 84.8 / 86.2.
struct Clip { const NormOut* clip; const double* part; int parts; double gscale, max_norm; float* norm_out; };
constexpr int FEW_PARTS = 1024;

template <bool GBF, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const dppm_tensor_entry* __restrict__ tab, const int2* __restrict__ chunks, Clip clip, StepArgs a) {
  const int2 ch = chunks[blockIdx.x];
  const dppm_tensor_entry e = tab[ch.x];
  float mult = a.gscale;
  if (clip.clip || clip.parts > 0) {
    const NormOut o = clip.clip ? *clip.clip : clip_of(clip.part, clip.parts, clip.gscale, clip.max_norm, blockIdx.x == 0 ? clip.norm_out : nullptr);
    if (!o.ok) return;
    mult = o.mult;
  }
  const long base = (long)ch.y * CHUNK;
  if (base + CHUNK <= e.numel) adamw_chunk<GBF, BITS, true>(e, base, (uint32_t)ch.x, mult, a);
  else adamw_chunk<GBF, BITS, false>(e, base, (uint32_t)ch.x, mult, a);
}

}  // namespace
}  // namespace dppm

using namespace dppm;

extern "C" int dppm_adamw_chunk(void) { return CHUNK; }

extern "C" size_t dppm_adamw_workspace_bytes(void) { return (NORM_GRID + 2) * sizeof(double); }

extern "C" int dppm_adamw_step(const dppm_tensor_entry* table, const int32_t* chunks, int n_chunks, int grad_bf16, int state_bits, double lr,
                               double beta1, double beta2, double eps, int step, double grad_scale, double max_norm, uint64_t seed,
                               float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  DPPM_REQUIRE(n_chunks >= 0 && step >= 1, "dppm_adamw_step: n_chunks=%d step=%d", n_chunks, step);
  DPPM_REQUIRE(state_bits == 8 || state_bits == 32, "dppm_adamw_step: state_bits=%d (8 or 32)", state_bits);
  DPPM_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0, "dppm_adamw_step: beta1=%g beta2=%g eps=%g", beta1, beta2, eps);
  DPPM_REQUIRE(n_chunks == 0 || (table && chunks), "dppm_adamw_step: null pointer");
  const bool clip = max_norm > 0;
  if (clip) {
    DPPM_REQUIRE(norm_out && workspace, "dppm_adamw_step: clipping needs norm_out and a workspace");
    DPPM_REQUIRE(workspace_bytes >= dppm_adamw_workspace_bytes(), "dppm_adamw_step: workspace of %zu bytes, %zu needed", workspace_bytes, dppm_adamw_workspace_bytes());
  }
  const hipStream_t st = as_stream(stream);
  const int2* ch = reinterpret_cast<const int2*>(chunks);
  Clip no{};
  if (clip) {
    double* part = reinterpret_cast<double*>(workspace);
    NormOut* out = reinterpret_cast<NormOut*>(part + NORM_GRID);
    // two chunks are read at a time: with few, two for each workgroup, so that the step can sum the parts itself
    const int grid = n_chunks <= 2 * FEW_PARTS ? (n_chunks + 1) / 2 : n_chunks < NORM_GRID ? n_chunks : NORM_GRID;
    if (grid > 0) {
      if (grad_bf16) hipLaunchKernelGGL((grad_sq_kernel<true>), dim3(grid), dim3(256), 0, st, table, ch, n_chunks, part);
      else hipLaunchKernelGGL((grad_sq_kernel<false>), dim3(grid), dim3(256), 0, st, table, ch, n_chunks, part);
    }
    if (grid > 0 && grid <= FEW_PARTS) {
      no.part = part; no.parts = grid; no.gscale = grad_scale; no.max_norm = max_norm; no.norm_out = norm_out;
    } else {
      hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, st, part, grid, grad_scale, max_norm, norm_out, out);
      no.clip = out;
    }
  }
  if (n_chunks > 0) {
    StepArgs a;
    a.one_minus_b1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.one_minus_b2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.step_size = (float)(lr / (1.0 - std::pow(beta1, step)));
    a.bc2_rsqrt = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, step)));
    a.gscale = (float)grad_scale;
    a.lr = lr;
    a.step = (uint32_t)step;
    a.key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const dim3 grid(n_chunks), block(256);
    if (grad_bf16) {
      if (state_bits == 8) hipLaunchKernelGGL((adamw_kernel<true, 8>), grid, block, 0, st, table, ch, no, a);
      else hipLaunchKernelGGL((adamw_kernel<true, 32>), grid, block, 0, st, table, ch, no, a);
    } else {
      if (state_bits == 8) hipLaunchKernelGGL((adamw_kernel<false, 8>), grid, block, 0, st, table, ch, no, a);
      else hipLaunchKernelGGL((adamw_kernel<false, 32>), grid, block, 0, st, table, ch, no, a);
    }
  }
  return check_launch("dppm_adamw_step");
}

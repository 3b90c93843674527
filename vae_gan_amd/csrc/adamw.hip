// AdamW over the flat buffer of an optimizer's tensors, states in 32 or in 8 bits.
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
// Tensors start at multiples of 256 elements; decay[block] says whether the tensor of that block is decayed.
// 8 bits: each block of 256 elements keeps m and r = sqrt(v) as e4m3 codes and one f32 scale each (largest magnitude / 448).
// The root halves the dynamic range that the codes have to span (e4m3 reaches 2^17.8 below its largest value, 2^35 in v); r is
// rounded to nearest but never down to 0, since an update divides by it.  The update uses this step's m and v before they
// are rounded.  A scale that follows the largest value (not a power of two) lets a block of unchanging codes decay.
// Bound by memory: 28 bytes a parameter at 32 bits, 16.06 at 8.
#include "common.h"
#include "rows.h"

#define ADAMW_BLOCK 256

struct AdamwParams {
  float *p;
  const float *g;
  const unsigned char *decay;
  int64_t blocks;
  float keep;          // 1 - lr wd, of decayed blocks
  float b1, b2, c1, c2;       // c = 1 - b
  float eps, step, rsqrt_bc2, gscale;
};

// one product and one sum each, never contracted: the state after a step is the same bits wherever it is computed
__device__ __forceinline__ void adamw_moments(float g, const AdamwParams& a, float& m, float& v) {
#pragma clang fp contract(off)
  m = m * a.b1 + g * a.c1;
  v = v * a.b2 + (g * g) * a.c2;
}
__device__ __forceinline__ float adamw_param(float p, float m, float root, float keep, const AdamwParams& a) {
#pragma clang fp contract(off)
  return p * keep - a.step * (m / (root * a.rsqrt_bc2 + a.eps));
}

__global__ __launch_bounds__(256) void adamw_kernel(const AdamwParams a, float* __restrict__ ms, float* __restrict__ vs) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t blk = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6); blk < a.blocks; blk += waves) {
    const int64_t o = blk * ADAMW_BLOCK + lane * 4;
    f32x4 p = *(const f32x4*)(a.p + o), g = *(const f32x4*)(a.g + o), m = *(const f32x4*)(ms + o), v = *(const f32x4*)(vs + o);
    const float keep = !a.decay || a.decay[blk] ? a.keep : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float mm = m[e], vv = v[e];
      adamw_moments(g[e] * a.gscale, a, mm, vv);
      m[e] = mm; v[e] = vv;
      p[e] = adamw_param(p[e], mm, sqrtf(vv), keep, a);
    }
    *(f32x4*)(a.p + o) = p;
    *(f32x4*)(ms + o) = m;
    *(f32x4*)(vs + o) = v;
  }
}

__device__ __forceinline__ float finite_abs(float v) { const float a = fabsf(v); return a < __builtin_inff() ? a : 0.f; }

// a wave's 256 values as e4m3 codes and their scale.  Values that are not finite get the NaN code and do not set the scale
// (the other elements of the block keep theirs).  The scale stays at least 2^-126, so its reciprocal is finite.
template <bool ROOT> __device__ __forceinline__ unsigned encode8(const f32x4& v, float& scale) {
  float most = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
  scale = fmaxf(wave_max64(most) * (1.f / 448.f), 0x1p-126f);
  const float inv = 1.f / scale;
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = v[e] * inv;
    if (ROOT && v[e] > 0.f) q[e] = fmaxf(q[e], 0x1p-9f);
    q[e] = fabsf(v[e]) < __builtin_inff() ? fminf(fmaxf(q[e], -448.f), 448.f) : __builtin_nanf("");
  }
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
}
__device__ __forceinline__ f32x4 decode8(unsigned c, float scale) {
  return f32x4{__builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale, __builtin_amdgcn_cvt_f32_fp8((int)c, 1) * scale,
               __builtin_amdgcn_cvt_f32_fp8((int)c, 2) * scale, __builtin_amdgcn_cvt_f32_fp8((int)c, 3) * scale};
}

__global__ __launch_bounds__(256) void adamw8_kernel(const AdamwParams a, unsigned* __restrict__ mc, float* __restrict__ mscale,
                                                     unsigned* __restrict__ rc, float* __restrict__ rscale) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t blk = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6); blk < a.blocks; blk += waves) {
    const int64_t o = blk * ADAMW_BLOCK + lane * 4;
    f32x4 p = *(const f32x4*)(a.p + o), g = *(const f32x4*)(a.g + o);
    f32x4 m = decode8(mc[o / 4], mscale[blk]), r = decode8(rc[o / 4], rscale[blk]);
    const float keep = !a.decay || a.decay[blk] ? a.keep : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float mm = m[e], vv = r[e] * r[e];
      adamw_moments(g[e] * a.gscale, a, mm, vv);
      m[e] = mm;
      r[e] = sqrtf(vv);
      p[e] = adamw_param(p[e], mm, r[e], keep, a);
    }
    *(f32x4*)(a.p + o) = p;
    float sm, sr;
    mc[o / 4] = encode8<false>(m, sm);
    rc[o / 4] = encode8<true>(r, sr);
    if (lane == 0) { mscale[blk] = sm; rscale[blk] = sr; }
  }
}

static int adamw_fill(const char* what, AdamwParams* a, float* p, const float* g, const unsigned char* decay, int64_t n, double lr,
                      double beta1, double beta2, double eps, double wd, int step, float grad_scale) {
  VG_REQUIRE(p && g && n > 0 && n % ADAMW_BLOCK == 0, "%s: null pointer, or a length %ld that is no multiple of %d", what, (long)n, ADAMW_BLOCK);
  VG_REQUIRE(((uintptr_t)p | (uintptr_t)g) % 16 == 0, "%s: buffers must be 16-byte aligned", what);
  VG_REQUIRE(step >= 1 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0 && wd >= 0,
             "%s: step %d, lr %g, betas %g %g, eps %g, weight decay %g", what, step, lr, beta1, beta2, eps, wd);
  // doubles: 1 - (float)0.999 is 1.3e-5 off 0.001
  const double bc1 = 1.0 - pow(beta1, step), bc2 = 1.0 - pow(beta2, step);
  *a = AdamwParams{p, g, decay, n / ADAMW_BLOCK, (float)(1.0 - lr * wd), (float)beta1, (float)beta2, (float)(1.0 - beta1),
                   (float)(1.0 - beta2), (float)eps, (float)(lr / bc1), (float)(1.0 / sqrt(bc2)), grad_scale};
  return VG_OK;
}
static unsigned adamw_grid(int64_t blocks) {
  const int64_t b = vg_ceil_div(blocks, 4);
  return (unsigned)(b < 8192 ? b : 8192);
}

extern "C" int vg_adamw_step(float* p, const float* g, float* m, float* v, const unsigned char* decay, int64_t n, double lr, double beta1,
                             double beta2, double eps, double weight_decay, int step, float grad_scale, void* stream) {
  AdamwParams a;
  if (int rc = adamw_fill("adamw_step", &a, p, g, decay, n, lr, beta1, beta2, eps, weight_decay, step, grad_scale)) return rc;
  VG_REQUIRE(m && v && ((uintptr_t)m | (uintptr_t)v) % 16 == 0, "adamw_step: states must be 16-byte aligned");
  hipLaunchKernelGGL(adamw_kernel, dim3(adamw_grid(a.blocks)), dim3(256), 0, (hipStream_t)stream, a, m, v);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

extern "C" int vg_adamw8_step(float* p, const float* g, void* m_codes, float* m_scale, void* r_codes, float* r_scale,
                              const unsigned char* decay, int64_t n, double lr, double beta1, double beta2, double eps, double weight_decay,
                              int step, float grad_scale, void* stream) {
  AdamwParams a;
  if (int rc = adamw_fill("adamw8_step", &a, p, g, decay, n, lr, beta1, beta2, eps, weight_decay, step, grad_scale)) return rc;
  VG_REQUIRE(m_codes && m_scale && r_codes && r_scale && ((uintptr_t)m_codes | (uintptr_t)r_codes) % 4 == 0,
             "adamw8_step: states must be 4-byte aligned");
  hipLaunchKernelGGL(adamw8_kernel, dim3(adamw_grid(a.blocks)), dim3(256), 0, (hipStream_t)stream, a, (unsigned*)m_codes, m_scale,
                     (unsigned*)r_codes, r_scale);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

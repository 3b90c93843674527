// AdamW over the flat buffer of an optimizer's tensors, states in 32 or in 8 bits.
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
// Tensors start at multiples of 256 elements; decay[block] says whether the tensor of that block is decayed.
// 8 bits: each block of 256 elements keeps m and r = sqrt(v) as e4m3 codes and one f32 scale each (largest magnitude / 448).
// The root halves the dynamic range that the codes have to span (e4m3 reaches 2^17.8 below its largest value, 2^35 in v); r is
// rounded to nearest but never down to 0, since an update divides by it.  The update uses this step's m and v before they
// are rounded.  A scale that follows the largest value (not a power of two) lets a block of unchanging codes decay.
// Rounded to nearest, a code alone does not follow its element: with b2 = 0.999 a step moves r by some 0.05 % and a code's half
// step is 3 to 6 %, so r keeps its place beside the block's largest.  Where half of a block's gradients grow three times, the
// other half's r is 2.3 times too large after 1000 steps and 2.7 after 3000 (medians).  Rounded up with the probability of the
// part that is cut off (DITHER), codes follow on average: medians within 1 % in both, single elements within 20 % of theirs (one
// standard deviation); 169 M elements: 515 us, 470 to nearest (the random bits).
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
  unsigned dither;            // of this step
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

// Where the buffers exceed the last-level cache (ADAMW_STREAM bytes) a wave takes U = 4 neighbouring blocks, all loads first,
// with loads and stores that do not allocate; otherwise one block, so that few elements still spread over the chip.  No loop:
// short workgroups keep the memory busier than resident ones.  169 M elements: 781 us (6.1 TB/s) against 1104 for resident
// workgroups and 860 for short ones of U = 1; 18 M elements, which stay cached: 73 us with U = 1, 82 the other way.
// 8-bit states, 169 M: 453 us (6.0 TB/s) against 606.
#define ADAMW_STREAM (256ll << 20)
template <bool STREAM, typename V> __device__ __forceinline__ V ld(const V* p) { return STREAM ? __builtin_nontemporal_load(p) : *p; }
template <bool STREAM, typename V> __device__ __forceinline__ void st(V* p, V v) {
  if (STREAM) __builtin_nontemporal_store(v, p); else *p = v;
}

template <int U, bool STREAM>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwParams a, float* __restrict__ ms, float* __restrict__ vs) {
  const int lane = threadIdx.x & 63;
  const int64_t b0 = (blockIdx.x * (int64_t)4 + (threadIdx.x >> 6)) * U;
  f32x4 p[U], g[U], m[U], v[U];
  float keep[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (b0 + u >= a.blocks) break;
    const int64_t o = (b0 + u) * ADAMW_BLOCK + lane * 4;
    g[u] = ld<STREAM>((const f32x4*)(a.g + o));
    p[u] = ld<STREAM>((const f32x4*)(a.p + o));
    m[u] = ld<STREAM>((const f32x4*)(ms + o));
    v[u] = ld<STREAM>((const f32x4*)(vs + o));
    keep[u] = !a.decay || a.decay[b0 + u] ? a.keep : 1.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (b0 + u >= a.blocks) break;
    const int64_t o = (b0 + u) * ADAMW_BLOCK + lane * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float mm = m[u][e], vv = v[u][e];
      adamw_moments(g[u][e] * a.gscale, a, mm, vv);
      m[u][e] = mm; v[u][e] = vv;
      p[u][e] = adamw_param(p[u][e], mm, sqrtf(vv), keep[u], a);
    }
    st<STREAM>((f32x4*)(a.p + o), p[u]);
    st<STREAM>((f32x4*)(ms + o), m[u]);
    st<STREAM>((f32x4*)(vs + o), v[u]);
  }
}

__device__ __forceinline__ float finite_abs(float v) { const float a = fabsf(v); return a < __builtin_inff() ? a : 0.f; }

// 32 bits of an element's step, from its place, its gradient and the step's number, so equal on every run that has the same ones.
// A round of shifts, exclusive ors and products with odd constants (leading digits of the golden ratio and of the root of 2) over
// the place of a lane's four elements, and one over each, after which every bit depends on all of the input.
__device__ __forceinline__ unsigned mix(unsigned x) {
  x = (x ^ x >> 16) * 0x9E3779B9u;
  x = (x ^ x >> 15) * 0x6A09E667u;
  return x ^ x >> 16;
}
// |q| <= 448 to one of its two e4m3 neighbours: 16 random bits are added below the three that stay.  Subnormals (steps of 2^-9)
// are shifted up by 2^-6, where steps are the same.
__device__ __forceinline__ float dithered(float q, unsigned r16) {
  const float a = fabsf(q), up = a < 0x1p-6f ? 0x1p-6f : 0.f;
  const float v = __uint_as_float((__float_as_uint(a + up) + (r16 << 4)) & 0xFFF00000u) - up;
  return copysignf(v, q);
}

// a wave's 256 values as e4m3 codes and their scale.  Values that are not finite get the NaN code and do not set the scale
// (the other elements of the block keep theirs).  The scale stays at least 2^-126, so its reciprocal is finite.
// random: 16 bits an element, in the low (m) or the high (r) half
template <bool ROOT, bool DITHER> __device__ __forceinline__ unsigned encode8(const f32x4& v, float& scale, const unsigned* random) {
  float most = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
  scale = fmaxf(wave_max64(most) * (1.f / 448.f), 0x1p-126f);
  const float inv = 1.f / scale;
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = v[e] * inv;
    if (ROOT && v[e] > 0.f) q[e] = fmaxf(q[e], 0x1p-9f);
    q[e] = fminf(fmaxf(q[e], -448.f), 448.f);
    if (DITHER) q[e] = dithered(q[e], ROOT ? random[e] >> 16 : random[e] & 0xFFFFu);
    if (!(fabsf(v[e]) < __builtin_inff())) q[e] = __builtin_nanf("");
  }
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
}
__device__ __forceinline__ f32x4 decode8(unsigned c, float scale) {
  return f32x4{__builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale, __builtin_amdgcn_cvt_f32_fp8((int)c, 1) * scale,
               __builtin_amdgcn_cvt_f32_fp8((int)c, 2) * scale, __builtin_amdgcn_cvt_f32_fp8((int)c, 3) * scale};
}

template <int U, bool STREAM, bool DITHER>
__global__ __launch_bounds__(256) void adamw8_kernel(const AdamwParams a, unsigned* __restrict__ mc, float* __restrict__ mscale,
                                                     unsigned* __restrict__ rc, float* __restrict__ rscale) {
  const int lane = threadIdx.x & 63;
  const int64_t b0 = (blockIdx.x * (int64_t)4 + (threadIdx.x >> 6)) * U;
  f32x4 p[U], g[U];
  unsigned cm[U], cr[U];
  float keep[U], sm[U], sr[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (b0 + u >= a.blocks) break;
    const int64_t o = (b0 + u) * ADAMW_BLOCK + lane * 4;
    g[u] = ld<STREAM>((const f32x4*)(a.g + o));
    p[u] = ld<STREAM>((const f32x4*)(a.p + o));
    cm[u] = ld<STREAM>(mc + o / 4);
    cr[u] = ld<STREAM>(rc + o / 4);
    sm[u] = mscale[b0 + u];
    sr[u] = rscale[b0 + u];
    keep[u] = !a.decay || a.decay[b0 + u] ? a.keep : 1.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (b0 + u >= a.blocks) break;
    const int64_t o = (b0 + u) * ADAMW_BLOCK + lane * 4;
    f32x4 m = decode8(cm[u], sm[u]), r = decode8(cr[u], sr[u]);
    unsigned random[4] = {};
    const unsigned place = DITHER ? mix((unsigned)(o >> 2) ^ a.dither) + (unsigned)(o >> 34) : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (DITHER) random[e] = mix((place + e) ^ __float_as_uint(g[u][e]));
      float mm = m[e], vv = r[e] * r[e];
      adamw_moments(g[u][e] * a.gscale, a, mm, vv);
      m[e] = mm;
      r[e] = sqrtf(vv);
      p[u][e] = adamw_param(p[u][e], mm, r[e], keep[u], a);
    }
    st<STREAM>((f32x4*)(a.p + o), p[u]);
    st<STREAM>(mc + o / 4, encode8<false, DITHER>(m, sm[u], random));
    st<STREAM>(rc + o / 4, encode8<true, DITHER>(r, sr[u], random));
    if (lane == 0) { mscale[b0 + u] = sm[u]; rscale[b0 + u] = sr[u]; }
  }
}

static int adamw_fill(const char* what, AdamwParams* a, float* p, const float* g, const unsigned char* decay, int64_t n, double lr,
                      double beta1, double beta2, double eps, double wd, int step, float grad_scale) {
  VG_REQUIRE(p && g && n > 0 && n % ADAMW_BLOCK == 0 && n < (1LL << 40), "%s: null pointer, or a length %ld that is no multiple of %d", what, (long)n, ADAMW_BLOCK);
  VG_REQUIRE(((uintptr_t)p | (uintptr_t)g) % 16 == 0, "%s: buffers must be 16-byte aligned", what);
  VG_REQUIRE(step >= 1 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0 && wd >= 0,
             "%s: step %d, lr %g, betas %g %g, eps %g, weight decay %g", what, step, lr, beta1, beta2, eps, wd);
  // doubles: 1 - (float)0.999 is 1.3e-5 off 0.001
  const double bc1 = 1.0 - pow(beta1, step), bc2 = 1.0 - pow(beta2, step);
  *a = AdamwParams{p, g, decay, n / ADAMW_BLOCK, (float)(1.0 - lr * wd), (float)beta1, (float)beta2, (float)(1.0 - beta1),
                   (float)(1.0 - beta2), (float)eps, (float)(lr / bc1), (float)(1.0 / sqrt(bc2)), grad_scale, (unsigned)step * 0x9E3779B9u};
  return VG_OK;
}
static dim3 adamw_grid(int64_t blocks, int u) { return dim3((unsigned)vg_ceil_div(blocks, 4 * u)); }

extern "C" int vg_adamw_step(float* p, const float* g, float* m, float* v, const unsigned char* decay, int64_t n, double lr, double beta1,
                             double beta2, double eps, double weight_decay, int step, float grad_scale, void* stream) {
  AdamwParams a;
  if (int rc = adamw_fill("adamw_step", &a, p, g, decay, n, lr, beta1, beta2, eps, weight_decay, step, grad_scale)) return rc;
  VG_REQUIRE(m && v && ((uintptr_t)m | (uintptr_t)v) % 16 == 0, "adamw_step: states must be 16-byte aligned");
  if (n * 28 > ADAMW_STREAM) hipLaunchKernelGGL((adamw_kernel<4, true>), adamw_grid(a.blocks, 4), dim3(256), 0, (hipStream_t)stream, a, m, v);
  else hipLaunchKernelGGL((adamw_kernel<1, false>), adamw_grid(a.blocks, 1), dim3(256), 0, (hipStream_t)stream, a, m, v);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

template <bool DITHER>
static int adamw8_launch(const char* what, float* p, const float* g, void* m_codes, float* m_scale, void* r_codes, float* r_scale,
                         const unsigned char* decay, int64_t n, double lr, double beta1, double beta2, double eps, double weight_decay,
                         int step, float grad_scale, hipStream_t st) {
  AdamwParams a;
  if (int rc = adamw_fill(what, &a, p, g, decay, n, lr, beta1, beta2, eps, weight_decay, step, grad_scale)) return rc;
  VG_REQUIRE(m_codes && m_scale && r_codes && r_scale && ((uintptr_t)m_codes | (uintptr_t)r_codes) % 4 == 0,
             "%s: states must be 4-byte aligned", what);
  if (n * 16 > ADAMW_STREAM)
    hipLaunchKernelGGL((adamw8_kernel<4, true, DITHER>), adamw_grid(a.blocks, 4), dim3(256), 0, st, a, (unsigned*)m_codes, m_scale,
                       (unsigned*)r_codes, r_scale);
  else
    hipLaunchKernelGGL((adamw8_kernel<1, false, DITHER>), adamw_grid(a.blocks, 1), dim3(256), 0, st, a, (unsigned*)m_codes, m_scale,
                       (unsigned*)r_codes, r_scale);
  VG_LAUNCH_CHECK();
  return VG_OK;
}
extern "C" int vg_adamw8_step(float* p, const float* g, void* m_codes, float* m_scale, void* r_codes, float* r_scale,
                              const unsigned char* decay, int64_t n, double lr, double beta1, double beta2, double eps, double weight_decay,
                              int step, float grad_scale, void* stream) {
  return adamw8_launch<false>("adamw8_step", p, g, m_codes, m_scale, r_codes, r_scale, decay, n, lr, beta1, beta2, eps, weight_decay, step,
                              grad_scale, (hipStream_t)stream);
}
extern "C" int vg_adamw8_dithered_step(float* p, const float* g, void* m_codes, float* m_scale, void* r_codes, float* r_scale,
                                       const unsigned char* decay, int64_t n, double lr, double beta1, double beta2, double eps,
                                       double weight_decay, int step, float grad_scale, void* stream) {
  return adamw8_launch<true>("adamw8_dithered_step", p, g, m_codes, m_scale, r_codes, r_scale, decay, n, lr, beta1, beta2, eps, weight_decay,
                             step, grad_scale, (hipStream_t)stream);
}

// y = act(x W^T + b) + res and its gradient, x [M][K] and W [N][K] row-major, bf16 or f32, accumulated in f32 on the matrix
// cores.  dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz;  dres = dy.  z = x W^T + b is stored beside y when a
// gradient will be wanted (act' of a stored z: one rounding of z to the storage type).
// All three products are C[i][j] = sum_k A(i, k) B(j, k) with element strides for i / j and k, so one kernel takes any of
// them, any alignment and any row stride.
#include "common.h"
#include "rows.h"

__device__ __forceinline__ float la_act(float z, int act) {
  switch (act) {
    case VG_ACT_LRELU: return z > 0.f ? z : VG_LRELU_SLOPE * z;
    case VG_ACT_SIGMOID: return 1.f / (1.f + __expf(-z));
    case VG_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case VG_ACT_SILU: return z / (1.f + __expf(-z));
    default: return z;
  }
}
__device__ __forceinline__ float la_slope(float z, int act) {
  switch (act) {
    case VG_ACT_LRELU: return z > 0.f ? 1.f : VG_LRELU_SLOPE;
    case VG_ACT_SIGMOID: { const float p = 1.f / (1.f + __expf(-z)); return p * (1.f - p); }
    case VG_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    case VG_ACT_SILU: { const float p = 1.f / (1.f + __expf(-z)); return p * (1.f + z * (1.f - p)); }
    default: return 1.f;
  }
}

struct GemmParams {
  const void *a, *b;
  int64_t ai, ak, bj, bk;       // element strides
  int m, n, k;
  void* c;                      // [m][n] out, row stride ldc
  int64_t ldc;
  int c_f32;                    // C is f32 although the operands are bf16 (gradient of an f32 master weight)
  const void* bias;             // [n] or null
  int bias_f32;
  const void* res;              // [m][n], row stride ldres, or null
  int64_t ldres;
  void* z;                      // [m][n] pre-activation out, or null
  int act;
};

template <typename T> __device__ __forceinline__ f32x4 la_mma(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 la_mma<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// a lane's 16 bytes are 4 k of its k-group: any assignment of k to the four products is right as long as A and B agree
template <> __device__ __forceinline__ f32x4 la_mma<float>(u32x4 a, u32x4 b, f32x4 c) {
  const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
  return c;
}

// one output element through the epilogue
template <typename T> __device__ __forceinline__ void la_store(const GemmParams& p, int i, int j, float v) {
  if (p.bias) v += p.bias_f32 ? ((const float*)p.bias)[j] : (float)((const T*)p.bias)[j];
  if (p.z) ((T*)p.z)[(int64_t)i * p.n + j] = (T)v;
  v = la_act(v, p.act);
  if (p.res) v += (float)((const T*)p.res)[(int64_t)i * p.ldres + j];
  if (p.c_f32) ((float*)p.c)[(int64_t)i * p.ldc + j] = v;
  else ((T*)p.c)[(int64_t)i * p.ldc + j] = (T)v;
}

// 64 x 64 tile, 4 waves of 32 x 32, 64 bytes of k a step, element loads with bounds
template <typename T> __global__ __launch_bounds__(256) void gemm_any_kernel(const GemmParams p) {
  constexpr int KT = 64 / sizeof(T), LD = KT + 16 / sizeof(T), PER = 64 * KT / 256;
  __shared__ __attribute__((aligned(16))) T sa[64 * LD], sb[64 * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tn = (p.n + 63) / 64;
  const int i0 = (int)(blockIdx.x / tn) * 64, j0 = (int)(blockIdx.x % tn) * 64;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  const T *A = (const T*)p.a, *B = (const T*)p.b;
  f32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < p.k; k0 += KT) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int q = tid + e * 256;
      // neighbouring threads take neighbouring memory
      const int ra = p.ak == 1 ? q / KT : q % 64, ka = p.ak == 1 ? q % KT : q / 64;
      const int rb = p.bk == 1 ? q / KT : q % 64, kb = p.bk == 1 ? q % KT : q / 64;
      sa[ra * LD + ka] = i0 + ra < p.m && k0 + ka < p.k ? A[(i0 + ra) * p.ai + (k0 + ka) * p.ak] : (T)0.f;
      sb[rb * LD + kb] = j0 + rb < p.n && k0 + kb < p.k ? B[(j0 + rb) * p.bj + (k0 + kb) * p.bk] : (T)0.f;
    }
    __syncthreads();
    const int off = (lane & 15) * LD + (lane >> 4) * (16 / (int)sizeof(T));
    u32x4 fa[2], fb[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      fa[u] = *(const u32x4*)(sa + (wi + u * 16) * LD + off);
      fb[u] = *(const u32x4*)(sb + (wj + u * 16) * LD + off);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) acc[u][v] = la_mma<T>(fa[u], fb[v], acc[u][v]);
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + wi + u * 16 + (lane >> 4) * 4 + r, j = j0 + wj + v * 16 + (lane & 15);
        if (i < p.m && j < p.n) la_store<T>(p, i, j, acc[u][v][r]);
      }
}

// dz = dy act'(z) and partial column sums of the unrounded dz: part[row chunk][n]
template <typename T>
__global__ __launch_bounds__(256) void la_dz_kernel(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                    float* __restrict__ part, int m, int n, int act, int rows_per) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  const int r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < m ? r0 + rows_per : m;
  float s = 0.f;
  for (int r = r0; r < r1; ++r) {
    const int64_t o = (int64_t)r * n + j;
    float g = (float)dy[o];
    if (act != VG_ACT_NONE) {
      g *= la_slope((float)z[o], act);
      dz[o] = (T)g;
    }
    s += g;
  }
  if (part) part[(int64_t)blockIdx.y * n + j] = s;
}

static int la_gemm(const GemmParams& p, int dtype, hipStream_t st) {
  const int64_t tiles = vg_ceil_div(p.n, 64) * vg_ceil_div(p.m, 64);
  VG_REQUIRE(tiles < (1LL << 31), "linear_act: %d x %d outputs are too many for one launch", p.m, p.n);
  const dim3 grid((unsigned)tiles);
  if (dtype == VG_BF16) hipLaunchKernelGGL(gemm_any_kernel<bf16_t>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(gemm_any_kernel<float>, grid, dim3(256), 0, st, p);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

static int la_check(const char* what, int64_t m, int64_t n, int64_t k, int act, int dtype) {
  VG_REQUIRE(dtype == VG_F32 || dtype == VG_BF16, "%s: dtype %d", what, dtype);
  VG_REQUIRE(m >= 1 && n >= 1 && k >= 1 && m < (1LL << 30) && n < (1LL << 22) && k < (1LL << 30), "%s: %ld x %ld x %ld", what, (long)m, (long)n, (long)k);
  VG_REQUIRE(act >= VG_ACT_NONE && act <= VG_ACT_SILU, "%s: activation %d", what, act);
  return VG_OK;
}

extern "C" int vg_linear_act_fwd(const void* x, int64_t ldx, const void* w, const void* bias, int bias_dtype, const void* res,
                                 int64_t ldres, void* y, void* z, int64_t m, int64_t n, int64_t k, int act, int dtype, void* stream) {
  if (int rc = la_check("linear_act_fwd", m, n, k, act, dtype)) return rc;
  VG_REQUIRE(x && w && y && ldx >= k && (!res || ldres >= n), "linear_act_fwd: null pointer or a short row stride");
  GemmParams p = {x, w, ldx, 1, k, 1, (int)m, (int)n, (int)k, y, n, 0, bias, bias_dtype == VG_F32, res, ldres, z, act};
  return la_gemm(p, dtype, (hipStream_t)stream);
}

static const int LA_DZ_PARTS = 256;
extern "C" size_t vg_linear_act_dz_ws_bytes(int64_t m, int64_t n) {
  return (size_t)(m < LA_DZ_PARTS ? m : LA_DZ_PARTS) * (size_t)n * sizeof(float);
}
extern "C" int vg_linear_act_dz(const void* dy, const void* z, void* dz, void* db, int bias_dtype, void* ws, int64_t m, int64_t n, int act,
                                int dtype, void* stream) {
  if (int rc = la_check("linear_act_dz", m, n, 1, act, dtype)) return rc;
  VG_REQUIRE(dy && (act == VG_ACT_NONE || (z && dz)) && (!db || ws), "linear_act_dz: null pointer");
  if (act == VG_ACT_NONE && !db) return VG_OK;
  hipStream_t st = (hipStream_t)stream;
  int parts = (int)(m < LA_DZ_PARTS ? m : LA_DZ_PARTS);
  const int per = (int)vg_ceil_div(m, parts);
  parts = (int)vg_ceil_div(m, per);
  const dim3 grid((unsigned)vg_ceil_div(n, 256), (unsigned)parts);
  float* part = db ? (float*)ws : nullptr;
  if (dtype == VG_BF16)
    hipLaunchKernelGGL(la_dz_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t*)dy, (const bf16_t*)z, (bf16_t*)dz, part, (int)m, (int)n, act, per);
  else hipLaunchKernelGGL(la_dz_kernel<float>, grid, dim3(256), 0, st, (const float*)dy, (const float*)z, (float*)dz, part, (int)m, (int)n, act, per);
  VG_LAUNCH_CHECK();
  if (db) return vg_fold_cols(part, parts, n, db, n, nullptr, bias_dtype, st);
  return VG_OK;
}

extern "C" int vg_linear_act_dgrad(const void* dz, const void* w, void* dx, int64_t m, int64_t n, int64_t k, int dtype, void* stream) {
  if (int rc = la_check("linear_act_dgrad", m, n, k, VG_ACT_NONE, dtype)) return rc;
  VG_REQUIRE(k < (1LL << 22) && dz && w && dx, "linear_act_dgrad: null pointer, or too wide");
  GemmParams p = {dz, w, n, 1, 1, k, (int)m, (int)k, (int)n, dx, k, 0, nullptr, 0, nullptr, 0, nullptr, VG_ACT_NONE};
  return la_gemm(p, dtype, (hipStream_t)stream);
}

extern "C" int vg_linear_act_wgrad(const void* dz, const void* x, int64_t ldx, void* dw, int dw_dtype, int64_t m, int64_t n, int64_t k,
                                   int dtype, void* stream) {
  if (int rc = la_check("linear_act_wgrad", m, n, k, VG_ACT_NONE, dtype)) return rc;
  VG_REQUIRE(k < (1LL << 22) && dz && x && dw && ldx >= k, "linear_act_wgrad: null pointer, a short row stride, or too wide");
  GemmParams p = {dz, x, 1, n, 1, ldx, (int)n, (int)k, (int)m, dw, k, dw_dtype == VG_F32, nullptr, 0, nullptr, 0, nullptr, VG_ACT_NONE};
  return la_gemm(p, dtype, (hipStream_t)stream);
}

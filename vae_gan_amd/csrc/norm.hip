// Layer norm over the last dimension, forward and backward, and the column reduction that its parameter gradients (and the
// bias gradient of vg_linear_act_dz) end in.
//   mu = sum x / c, var = sum (x - mu)^2 / c, r = (var + eps)^-1/2, xh = (x - mu) r, y = xh w + b
//   g = dy w:  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
// Rows are [c valid + padding] elements with a row stride; padding columns of y / dx are written as zeros (the NHWC
// convention).  Bound by memory: x is read and y written once; backward reads x and dy and writes dx once.  A row is held
// in the registers of GL lanes (a part of a wave, a wave, or the block's four waves) as NV accesses of VEC elements, so the
// variance is that of the centred values (no cancellation of sum(x^2) - mu^2) at no second read.  All sums are f32; the mean of
// the centred values, which is what the first mean's rounding left in them, is taken off them again: constant rows are exactly
// centred and y = b, where a mean one step off would be raised by r, up to 316 at eps = 1e-5.
// 16384 x 512 bf16: forward 10.3 us alone (3.3 TB/s; 9.4 without the second mean), 11.6 in a training pass, backward 13.5 us (3.7
// TB/s) and 3.9 us for the column sums; 65536 x 128 f32 forward 14.8 us (4.5 TB/s; 13.6), where the launch's own few us weigh less.
#include "common.h"
#include "rows.h"

// VEC elements as loaded, so that the next row can be on its way while this one is worked on.  Accesses are aligned to an element
// only (rows of any stride; the machine's global memory instructions take that).  PART: the last one of a row may have n < VEC
// elements; whole rows do not pay for that (1024 x 8192 f32 forward: 17.1 us with, 13.4 without; x 8191 by elements: 26, so 17.1).
template <typename T, int VEC, bool PART> struct Raw {
  typedef T vt __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  T __attribute__((ext_vector_type(VEC))) v;
  __device__ __forceinline__ void load(const T* p, int n) {
    if (!PART || n >= VEC) v = *(const vt*)p;
    else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = e < n ? p[e] : (T)0.f;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (T)0.f;
  }
  __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
};
// a lane's parameters, zero past c; 16-byte loads where the lane's columns allow them
template <int VEC> __device__ __forceinline__ void ld_param(const float* w, int col, int c, float* o) {
  if (VEC % 4 == 0 && col + VEC <= c && (uintptr_t)w % 16 == 0) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const f32x4 q = *(const f32x4*)(w + col + e);
#pragma unroll
      for (int i = 0; i < (VEC < 4 ? VEC : 4); ++i) o[e + i] = q[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = col + e < c ? w[col + e] : 0.f;
  }
}
template <typename T, int VEC, bool PART> __device__ __forceinline__ void st_vec(T* p, const float* o, int n) {
  typedef T vt __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  if (!PART || n >= VEC) {
    vt v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (T)o[e];
    *(vt*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < n) p[e] = (T)o[e];
  }
}

// sum over the GL lanes that share a row; every lane gets it.  GL == 256: through LDS (red: one slot per wave and value)
template <int GL> __device__ __forceinline__ float lane_sum(float v) {
  if constexpr (GL >= 64) v = wave_sum64(v);
  else {
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  }
  return v;
}
template <int GL> __device__ __forceinline__ float row_sum(float v, float* red, int slot) {
  v = lane_sum<GL>(v);
  if constexpr (GL > 64) {
    if ((threadIdx.x & 63) == 0) red[slot * 4 + (threadIdx.x >> 6)] = v;
    __syncthreads();
    v = (red[slot * 4] + red[slot * 4 + 1]) + (red[slot * 4 + 2] + red[slot * 4 + 3]);
  }
  return v;
}
// a product as one f32, not contracted into the differences that take it: those of equal values have to be equal and short
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
// two sums with one barrier between them, in slots `slot` and `slot` + 1
template <int GL> __device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int slot) {
  a = lane_sum<GL>(a);
  b = lane_sum<GL>(b);
  if constexpr (GL > 64) {
    if ((threadIdx.x & 63) == 0) { red[slot * 4 + (threadIdx.x >> 6)] = a; red[slot * 4 + 4 + (threadIdx.x >> 6)] = b; }
    __syncthreads();
    a = (red[slot * 4] + red[slot * 4 + 1]) + (red[slot * 4 + 2] + red[slot * 4 + 3]);
    b = (red[slot * 4 + 4] + red[slot * 4 + 5]) + (red[slot * 4 + 6] + red[slot * 4 + 7]);
  }
}

template <typename T, int VEC, int GL, int NV, bool PART>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                     const float* __restrict__ b, T* __restrict__ y, int64_t ldy,
                                                     float* __restrict__ stats, int64_t rows, int c, int cs, float eps) {
  __shared__ float red[24];
  constexpr int RPB = 256 / GL;
  const int gl = threadIdx.x % GL;
  const float n = (float)c, inv = 1.f / n;
  float wv[NV][VEC], bv[NV][VEC];                    // zero in the padding: y comes out as 0 there
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ld_param<VEC>(w, (i * GL + gl) * VEC, c, wv[i]);
    ld_param<VEC>(b, (i * GL + gl) * VEC, c, bv[i]);
  }
  Raw<T, VEC, PART> in[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GL + gl) * VEC;
      if (row < rows && col < cs) in[i].load(x + row * ldx + col, cs - col); else in[i].zero();
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int turn = 0;
  fetch(blockIdx.x * (int64_t)RPB + threadIdx.x / GL);
  for (int64_t r0 = blockIdx.x * (int64_t)RPB; r0 < rows; r0 += step, turn ^= 3) {
    const int64_t row = r0 + threadIdx.x / GL;
    const bool live = row < rows;                     // dead groups still take part in the shuffles and barriers
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = (i * GL + gl) * VEC + e < c ? in[i].get(e) : 0.f;
        s += v[i][e];
      }
    fetch(row + step);
    const float mu = rounded_product(row_sum<GL>(s, red, turn), inv);
    float q = 0.f, rest = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = (i * GL + gl) * VEC + e < c ? v[i][e] - mu : 0.f;
        rest += v[i][e];
        q += v[i][e] * v[i][e];
      }
    row_sum2<GL>(rest, q, red, turn + 1);
    rest /= n;                                       // divided: exact for a constant row
    const float r = 1.f / sqrtf(fmaxf((q - rest * rest * n) * inv, 0.f) + eps);
    if (!live) continue;
    if (stats && gl == 0) { stats[2 * row] = mu + rest; stats[2 * row + 1] = r; }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GL + gl) * VEC;
      if (col >= cs) break;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = col + e < c ? (v[i][e] - rest) * r * wv[i][e] + bv[i][e] : 0.f;
      st_vec<T, VEC, PART>(y + row * ldy + col, o, cs - col);
    }
  }
}

// rows too long for the registers of a block: three passes over the row (the second and third come from the caches)
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_long_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                          const float* __restrict__ b, T* __restrict__ y, int64_t ldy,
                                                          float* __restrict__ stats, int c, int cs, float eps) {
  __shared__ float red[12];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  float s = 0.f;
  for (int i = threadIdx.x; i < c; i += 256) s += (float)xr[i];
  const float mu = row_sum<256>(s, red, 0) / (float)c;
  float q = 0.f, rest = 0.f;
  for (int i = threadIdx.x; i < c; i += 256) { const float d = (float)xr[i] - mu; rest += d; q += d * d; }
  row_sum2<256>(rest, q, red, 1);
  rest /= (float)c;
  const float r = 1.f / sqrtf(fmaxf(q / (float)c - rest * rest, 0.f) + eps);
  if (stats && threadIdx.x == 0) { stats[2 * row] = mu + rest; stats[2 * row + 1] = r; }
  for (int i = threadIdx.x; i < cs; i += 256) y[row * ldy + i] = (T)(i < c ? ((float)xr[i] - mu - rest) * r * w[i] + b[i] : 0.f);
}

// dx of the rows of this block (block-strided; null: not wanted), and the block's partial sums of dw and db: part[block][2][c]
template <typename T, int VEC, int GL, int NV, bool PART>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                     const float* __restrict__ w, const float* __restrict__ stats,
                                                     T* __restrict__ dx, int64_t lddx, float* __restrict__ part, int64_t rows,
                                                     int c, int cs) {
  __shared__ float red[16];
  extern __shared__ float fold[];                    // [waves][GL x VEC] for the last fold (GL <= 64)
  constexpr int RPB = 256 / GL;
  const int gl = threadIdx.x % GL;
  const float inv = 1.f / (float)c;
  float aw[NV][VEC], ab[NV][VEC], wv[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    ld_param<VEC>(w, (i * GL + gl) * VEC, c, wv[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) aw[i][e] = ab[i][e] = 0.f;
  }
  Raw<T, VEC, PART> nx[NV], ng[NV];
  float nmu, nr;
  auto fetch = [&](int64_t row) {
    const bool live = row < rows;
    nmu = live ? stats[2 * row] : 0.f;
    nr = live ? stats[2 * row + 1] : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GL + gl) * VEC;
      if (live && col < cs) { nx[i].load(x + row * ldx + col, cs - col); ng[i].load(dy + row * lddy + col, cs - col); }
      else { nx[i].zero(); ng[i].zero(); }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int turn = 0;
  fetch(blockIdx.x * (int64_t)RPB + threadIdx.x / GL);
  for (int64_t r0 = blockIdx.x * (int64_t)RPB; r0 < rows; r0 += step, turn ^= 2) {
    const int64_t row = r0 + threadIdx.x / GL;
    const bool live = row < rows;
    float xh[NV][VEC], g[NV][VEC];
    const float mu = nmu, r = nr;
    float sg = 0.f, sgx = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) { xh[i][e] = nx[i].get(e); g[i][e] = ng[i].get(e); }
    fetch(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * GL + gl) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool in = live && col + e < c;
        xh[i][e] = in ? (xh[i][e] - mu) * r : 0.f;
        g[i][e] = in ? g[i][e] : 0.f;
        aw[i][e] += g[i][e] * xh[i][e];
        ab[i][e] += g[i][e];
        g[i][e] *= wv[i][e];
        sg += g[i][e];
        sgx += g[i][e] * xh[i][e];
      }
    }
    // two LDS slots in turn: a wave can be one row ahead of the readers of the other pair
    const float mg = row_sum<GL>(sg, red, turn) * inv, mgx = row_sum<GL>(sgx, red, turn + 1) * inv;
    if (live && dx) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * GL + gl) * VEC;
        if (col >= cs) break;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = col + e < c ? r * (g[i][e] - mg - xh[i][e] * mgx) : 0.f;
        st_vec<T, VEC, PART>(dx + row * lddx + col, o, cs - col);
      }
    }
  }
  if (!part) return;
  float* pw = part + (size_t)blockIdx.x * 2 * c;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int col = (i * GL + gl) * VEC + e;
      float a = aw[i][e], d = ab[i][e];
      if constexpr (GL < 64) {
#pragma unroll
        for (int o = GL; o < 64; o <<= 1) { a += __shfl_xor(a, o, 64); d += __shfl_xor(d, o, 64); }
      }
      if constexpr (GL <= 64) {                      // fold the block's four waves in a fixed order
        __syncthreads();
        if ((threadIdx.x & 63) < GL) { fold[(threadIdx.x >> 6) * GL + gl] = a; fold[(4 + (threadIdx.x >> 6)) * GL + gl] = d; }
        __syncthreads();
        if (threadIdx.x < GL && col < c) {
          pw[col] = (fold[gl] + fold[GL + gl]) + (fold[2 * GL + gl] + fold[3 * GL + gl]);
          pw[c + col] = (fold[4 * GL + gl] + fold[5 * GL + gl]) + (fold[6 * GL + gl] + fold[7 * GL + gl]);
        }
      } else if (col < c) { pw[col] = a; pw[c + col] = d; }
    }
}

// long rows: dx row by row; the parameter gradients by columns in a kernel of their own
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_long_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy,
                                                          const float* __restrict__ w, const float* __restrict__ stats,
                                                          T* __restrict__ dx, int64_t lddx, int c, int cs) {
  __shared__ float red[8];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * ldx, *dr = dy + row * lddy;
  const float mu = stats[2 * row], r = stats[2 * row + 1];
  float sg = 0.f, sgx = 0.f;
  for (int i = threadIdx.x; i < c; i += 256) {
    const float g = (float)dr[i] * w[i];
    sg += g;
    sgx += g * (((float)xr[i] - mu) * r);
  }
  const float mg = row_sum<256>(sg, red, 0) / (float)c, mgx = row_sum<256>(sgx, red, 1) / (float)c;
  for (int i = threadIdx.x; i < cs; i += 256)
    dx[row * lddx + i] = (T)(i < c ? r * ((float)dr[i] * w[i] - mg - ((float)xr[i] - mu) * r * mgx) : 0.f);
}
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_long_params_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                                 int64_t lddy, const float* __restrict__ stats,
                                                                 float* __restrict__ part, int64_t rows, int c, int64_t rows_per) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= c) return;
  const int64_t r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < rows ? r0 + rows_per : rows;
  float a = 0.f, d = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = (float)dy[r * lddy + col];
    a += g * (((float)x[r * ldx + col] - stats[2 * r]) * stats[2 * r + 1]);
    d += g;
  }
  part[(size_t)blockIdx.y * 2 * c + col] = a;
  part[(size_t)blockIdx.y * 2 * c + c + col] = d;
}

// out[col] = sum over parts of part[p][col]: 32 interleaved chains of parts a column, then the chains in order
template <typename O>
__global__ __launch_bounds__(1024) void fold_cols_kernel(const float* __restrict__ part, int parts, int64_t cols, O* __restrict__ out0,
                                                         int64_t split, O* __restrict__ out1) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, py = threadIdx.x >> 5;
  const int64_t col = blockIdx.x * (int64_t)32 + cx;
  float a = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int p = py; p < parts; p += 32) a += part[p * cols + col];
  }
  s[py][cx] = a;
  __syncthreads();
  if (py == 0 && col < cols) {
    float t = s[0][cx];
#pragma unroll
    for (int i = 1; i < 32; ++i) t += s[i][cx];
    O* o = col < split ? out0 + col : out1 + (col - split);
    if (col < split ? out0 != nullptr : out1 != nullptr) *o = (O)t;
  }
}

int vg_fold_cols(const float* part, int parts, int64_t cols, void* out0, int64_t split, void* out1, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)vg_ceil_div(cols, 32));
  if (dtype == VG_BF16)
    hipLaunchKernelGGL(fold_cols_kernel<bf16_t>, grid, dim3(1024), 0, st, part, parts, cols, (bf16_t*)out0, split, (bf16_t*)out1);
  else hipLaunchKernelGGL(fold_cols_kernel<float>, grid, dim3(1024), 0, st, part, parts, cols, (float*)out0, split, (float*)out1);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

// ---- host ----------------------------------------------------------------------------------------------------------
static const int64_t LN_FWD_BLOCKS = 1024, LN_BWD_BLOCKS = 768;
// blocks of the backward pass: enough to fill the chip, few enough that the partial sums (8 c bytes a block) stay small
static int64_t ln_bwd_blocks(int64_t rows, int rpb) {
  const int64_t need = vg_ceil_div(rows, rpb);
  return need < LN_BWD_BLOCKS ? need : LN_BWD_BLOCKS;
}
// forward: a block keeps the weights of its columns over several rows
static int64_t ln_fwd_blocks(int64_t rows, int rpb) {
  const int64_t need = vg_ceil_div(rows, rpb);
  return need < LN_FWD_BLOCKS ? need : LN_FWD_BLOCKS;
}
static const int LN_LONG_PARTS = 64;

struct LnArgs {
  const void *x, *dy;
  int64_t ldx, lddy, ldo;
  const float *w, *b;
  void* out;
  float *stats, *part;
  int64_t rows;
  int c, cs;
  float eps;
};

template <typename T, int VEC, int GL, int NV, bool PART> static void ln_launch(const LnArgs& a, bool bwd, hipStream_t st) {
  constexpr int RPB = 256 / GL;
  if (!bwd)
    hipLaunchKernelGGL((ln_fwd_kernel<T, VEC, GL, NV, PART>), dim3((unsigned)ln_fwd_blocks(a.rows, RPB)), dim3(256), 0, st, (const T*)a.x,
                       a.ldx, a.w, a.b, (T*)a.out, a.ldo, a.stats, a.rows, a.c, a.cs, a.eps);
  else
    hipLaunchKernelGGL((ln_bwd_kernel<T, VEC, GL, NV, PART>), dim3((unsigned)ln_bwd_blocks(a.rows, RPB)), dim3(256),
                       GL <= 64 ? 8 * GL * sizeof(float) : 0, st, (const T*)a.x, a.ldx, (const T*)a.dy, a.lddy, a.w, a.stats,
                       (T*)a.out, a.ldo, a.part, a.rows, a.c, a.cs);
}

// The lanes that share a row: the fewest whose VEC-element accesses cover it, so that narrow rows (a 41-channel latent) do
// not leave most of a wave idle; from one wave up the accesses per lane grow first (no barrier), then the whole block.
// Returns the number of parts, 0 for rows that do not fit (the long kernels).
template <typename T, bool PART> static int ln_dispatch_t(const LnArgs& a, bool bwd, hipStream_t st) {
  constexpr int VEC = Elt<T>::PIECE;
  const int n = (int)vg_ceil_div(a.cs, VEC);          // accesses a row needs
#define LN_CASE(GL, NV)                                                   \
  if (n <= GL * NV) {                                                     \
    ln_launch<T, VEC, GL, NV, PART>(a, bwd, st);                          \
    return (int)ln_bwd_blocks(a.rows, 256 / GL);                          \
  }
  LN_CASE(8, 1) LN_CASE(16, 1) LN_CASE(32, 1) LN_CASE(64, 1) LN_CASE(64, 2) LN_CASE(64, 4)
  if constexpr (VEC == 4) { LN_CASE(64, 8) LN_CASE(256, 4) LN_CASE(256, 8) }
  else { LN_CASE(256, 2) LN_CASE(256, 4) }
#undef LN_CASE
  return 0;
}
static int ln_dispatch(const LnArgs& a, int dtype, bool bwd, hipStream_t st) {
  if (dtype == VG_BF16) return a.cs % 8 ? ln_dispatch_t<bf16_t, true>(a, bwd, st) : ln_dispatch_t<bf16_t, false>(a, bwd, st);
  return a.cs % 4 ? ln_dispatch_t<float, true>(a, bwd, st) : ln_dispatch_t<float, false>(a, bwd, st);
}

static int ln_check(const char* what, int64_t rows, int c, int cs, int64_t ld0, int64_t ld1, int dtype) {
  VG_REQUIRE(dtype == VG_F32 || dtype == VG_BF16, "%s: dtype %d", what, dtype);
  VG_REQUIRE(rows >= 0 && rows < (1LL << 31) && c >= 1 && cs >= c && cs <= (1 << 24), "%s: %ld rows of %d columns, %d stored", what, (long)rows, c, cs);
  VG_REQUIRE(ld0 >= cs && ld1 >= cs, "%s: a row stride below the row's %d columns", what, cs);
  return VG_OK;
}

extern "C" int vg_layer_norm_fwd(const void* x, int64_t ldx, const float* w, const float* b, void* y, int64_t ldy, float* stats,
                                 int64_t rows, int c, int cs, float eps, int dtype, void* stream) {
  if (int rc = ln_check("layer_norm_fwd", rows, c, cs, ldx, ldy, dtype)) return rc;
  if (rows == 0) return VG_OK;
  VG_REQUIRE(x && w && b && y, "layer_norm_fwd: null pointer");
  VG_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps %g", (double)eps);
  hipStream_t st = (hipStream_t)stream;
  LnArgs a = {x, nullptr, ldx, 0, ldy, w, b, y, stats, nullptr, rows, c, cs, eps};
  if (!ln_dispatch(a, dtype, false, st)) {
    VG_GRID_CHECK("layer_norm_fwd", rows, 256);
    if (dtype == VG_BF16)
      hipLaunchKernelGGL(ln_fwd_long_kernel<bf16_t>, dim3((unsigned)rows), dim3(256), 0, st, (const bf16_t*)x, ldx, w, b, (bf16_t*)y, ldy, stats, c, cs, eps);
    else hipLaunchKernelGGL(ln_fwd_long_kernel<float>, dim3((unsigned)rows), dim3(256), 0, st, (const float*)x, ldx, w, b, (float*)y, ldy, stats, c, cs, eps);
  }
  VG_LAUNCH_CHECK();
  return VG_OK;
}

extern "C" size_t vg_layer_norm_bwd_ws_bytes(int64_t rows, int c) {
  // the most blocks any variant launches; long rows use LN_LONG_PARTS
  int64_t parts = rows < LN_BWD_BLOCKS ? rows : LN_BWD_BLOCKS;
  if (parts < LN_LONG_PARTS) parts = LN_LONG_PARTS;
  return (size_t)parts * 2 * (size_t)c * sizeof(float);
}

extern "C" int vg_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t lddy, const float* w, const float* stats,
                                 void* dx, int64_t lddx, float* dw, float* db, void* ws, int64_t rows, int c, int cs, int dtype,
                                 void* stream) {
  if (int rc = ln_check("layer_norm_bwd", rows, c, cs, ldx, lddy, dtype)) return rc;
  VG_REQUIRE(!dx || lddx >= cs, "layer_norm_bwd: a row stride below the row's %d columns", cs);
  VG_REQUIRE(rows > 0 && x && dy && w && stats && (dx || dw || db), "layer_norm_bwd: null pointer or no rows");
  VG_REQUIRE((!dw && !db) || ws, "layer_norm_bwd: the parameter gradients need a workspace");
  hipStream_t st = (hipStream_t)stream;
  float* part = dw || db ? (float*)ws : nullptr;
  LnArgs a = {x, dy, ldx, lddy, lddx, w, nullptr, dx, (float*)stats, part, rows, c, cs, 0.f};
  int parts = ln_dispatch(a, dtype, true, st);
  if (!parts) {
    VG_GRID_CHECK("layer_norm_bwd", rows, 256);
    parts = rows < LN_LONG_PARTS ? (int)rows : LN_LONG_PARTS;
    const int64_t per = vg_ceil_div(rows, parts);
    parts = (int)vg_ceil_div(rows, per);
    const dim3 grid((unsigned)vg_ceil_div(c, 256), (unsigned)parts);
    if (dtype == VG_BF16) {
      if (dx) hipLaunchKernelGGL(ln_bwd_long_kernel<bf16_t>, dim3((unsigned)rows), dim3(256), 0, st, (const bf16_t*)x, ldx, (const bf16_t*)dy, lddy, w, stats, (bf16_t*)dx, lddx, c, cs);
      if (part) hipLaunchKernelGGL(ln_bwd_long_params_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t*)x, ldx, (const bf16_t*)dy, lddy, stats, part, rows, c, per);
    } else {
      if (dx) hipLaunchKernelGGL(ln_bwd_long_kernel<float>, dim3((unsigned)rows), dim3(256), 0, st, (const float*)x, ldx, (const float*)dy, lddy, w, stats, (float*)dx, lddx, c, cs);
      if (part) hipLaunchKernelGGL(ln_bwd_long_params_kernel<float>, grid, dim3(256), 0, st, (const float*)x, ldx, (const float*)dy, lddy, stats, part, rows, c, per);
    }
  }
  VG_LAUNCH_CHECK();
  if (part) return vg_fold_cols(part, parts, 2 * (int64_t)c, dw, c, db, VG_F32, st);
  return VG_OK;
}

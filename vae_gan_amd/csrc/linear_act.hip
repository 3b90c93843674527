// y = act(x W^T + b) + res and its gradient, x [M][K] and W [N][K] row-major, bf16 or f32, accumulated in f32 on the matrix
// cores.  dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz;  dres = dy.
// The forward stores act'(z) beside y when a gradient will be wanted.  For bf16 tensors 2^14 act'(z) in f16: at most 2^-11
// relative, where a z or a slope rounded to bf16 would add an error as large as the gradient's own rounding; the factor (slopes
// are below 1.2, f16 ends at 65504) keeps that accuracy down to slopes of 2^-28, and anything above 2^-39 from becoming 0
// (a sigmoid or SiLU at z = -26; beside bf16 gradients, whose own range is longer, smaller ones are lost).
// dz is rounded to x's type before the two products of the backward pass, since bf16 matrix instructions take nothing wider:
// dx and dW of 16384 x 1024 x 4096 are off by 2.4e-3 of their size where their own rounding alone gives 1.7e-3.
// All three products are C[i][j] = sum_k A(i, k) B(j, k), each operand either with k contiguous (x, W, dz in the first two)
// or with i / j contiguous (W in dx = dz W, both in dW): a tile of the first kind is read from LDS with 16-byte reads, one of
// the second with transposing reads, so nothing is transposed in memory.
// Bound by the matrix cores where the sizes fill the chip (bf16 16384 x 1024 x 4096 in a training pass: forward 157 us without an
// activation, dx 116, dW 114 and 14 to join four parts: 875, 1180 and 1200 TFLOP/s), by launches and latency below some 10 GFLOP.
#include <type_traits>

#include "common.h"
#include "rows.h"

typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef _Float16 f16_t;

// e^x for x <= 0.  Beside f32 results the part of x log2 e that its f32 product leaves out is applied to the machine's base-2
// exponential (off by an ulp, as its reciprocal is), which is then off by 3 u instead of |x| u; beside bf16 that does not show.
// Below 2^-126 it is 0.
template <typename T> __device__ __forceinline__ float la_exp(float x) {
  constexpr float L = 1.4426950408889634f, L_REST = 1.92596299e-8f;      // log2 e
  if constexpr (sizeof(T) == 2) return __expf(x);
  x = x < -128.f ? -128.f : x;                       // a NaN stays one, and -inf does not make one
  const float h = x * L, rest = fmaf(x, L_REST, fmaf(x, L, -h)), e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, rest * 0.6931471805599453f, e);
}
// Phi(-|x|) = e^(-x^2/2) t P(t) with t = 1 / (1 + p |x|), and that exponential, which the density needs too.  P is fitted to the
// smallest relative error over |x| <= 13.5 (e^(-x^2/2) is 0 in f32 from there on), so z Phi(z) keeps its leading digits in the
// negative tail: 3.7e-6 of Phi with six coefficients, for results in bf16 (2^-9), 6.1e-8 with eight, for f32, where x^2 is
// carried in two parts as well.  A library erf costs four times the instructions, and 67 M of them took as long as the
// product of 16384 x 1024 x 4096 itself.
template <typename T> __device__ __forceinline__ float la_phi(float x, float& e) {
  const float a = fabsf(x), h = x * x;
  if constexpr (sizeof(T) == 2) {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.307628282f * a);
    e = la_exp<T>(-0.5f * h);
    return e * t * (0.122990536f + t * (0.118537826f + t * (0.137324485f + t * (0.00529493169f + t * (0.191671309f + t * -0.0758208932f)))));
  } else {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.305121229f * a), low = h < __builtin_inff() ? fmaf(x, x, -h) : 0.f;
    e = la_exp<T>(-0.5f * h);
    e -= e * 0.5f * low;
    return e * t * (0.121686477f + t * (0.122538544f + t * (0.103320019f + t * (0.121442011f + t * (-0.0387208932f +
           t * (0.186413127f + t * (-0.153564337f + t * 0.0368851234f)))))));
  }
}
// p = 1 / (1 + e^-x) and q = 1 - p, both from e^-|x| in (0, 1]: neither is a difference, so p's slope p q keeps its leading
// digits on either side.
template <typename T> __device__ __forceinline__ void la_logistic(float x, float& p, float& q) {
  const float e = la_exp<T>(-fabsf(x)), t = __builtin_amdgcn_rcpf(1.f + e);
  p = x < 0.f ? e * t : t;
  q = x < 0.f ? t : e * t;
}
// act(z) and act'(z), sharing the exponential
template <typename T, int N> __device__ __forceinline__ void la_act(float* z, int act, float* s) {
  switch (act) {                                     // one branch for all N: their exponentials overlap
    case VG_ACT_LRELU:
#pragma unroll
      for (int i = 0; i < N; ++i) { s[i] = z[i] > 0.f ? 1.f : VG_LRELU_SLOPE; z[i] *= s[i]; }
      break;
    case VG_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float p, q;
        la_logistic<T>(z[i], p, q);
        z[i] = p;
        s[i] = p * q;
      }
      break;
    case VG_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = z[i];
        float e;
        const float q = la_phi<T>(x, e), phi = x < 0.f ? q : 1.f - q;
        z[i] = x * phi;
        s[i] = phi + x * e * 0.39894228040143268f;
      }
      break;
    case VG_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = z[i];
        float p, q;
        la_logistic<T>(x, p, q);
        z[i] = x * p;
        s[i] = p * (1.f + x * q);
      }
      break;
    default: break;
  }
}

struct GemmParams {
  const void *a, *b;
  int64_t lda, ldb;             // elements between rows of the stored matrix ([m][k] or, transposed, [k][m])
  int m, n, k;
  void* c;                      // [m][n] out, row stride n
  int c_f32;                    // C is f32 although the operands are bf16 (gradient of an f32 master weight)
  const void* bias;             // [n] or null
  int bias_f32;
  const void* res;              // [m][n], row stride ldres, or null
  int64_t ldres;
  void* slope;                  // [m][n] act'(z) out (f16, 2^14 times, for bf16; f32 for f32), or null
  int act;
  float* part;                  // split k: [splits][m][ldp] f32 partial sums instead of C
  int splits, ldp, ktiles;      // ktiles: of one split
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

// ---- epilogue: eight neighbouring sums of row i, columns j.. -----------------------------------------------------------
template <typename T> struct SlopeT;
template <> struct SlopeT<bf16_t> { typedef f16_t type; static constexpr float ONE = 0x1p14f; };      // how a slope of 1 is kept
template <> struct SlopeT<float> { typedef float type; static constexpr float ONE = 1.f; };
// Rows of any length and stride: 16-byte accesses that are aligned to an element only, which this machine's global memory
// instructions take (f32 1001 x 515 x 1037 with SiLU, slopes and a residual: 37.5 us by elements, 32.8 so;
// bf16 16383 x 1024 x 4095 with GELU, slopes and a residual 385, 245).
template <typename O> __device__ __forceinline__ void put8(O* p, const float* v) {
  typedef O vt __attribute__((ext_vector_type(8), aligned(sizeof(O))));
  vt o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (O)v[e];
  *(vt*)p = o;
}
// for what is not read again soon
template <typename O> __device__ __forceinline__ void get8_nt(const O* p, float* v) {
  typedef O vt __attribute__((ext_vector_type(8), aligned(sizeof(O))));
  const vt o = __builtin_nontemporal_load((const vt*)p);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)o[e];
}
template <typename O> __device__ __forceinline__ void get8(const O* p, float* v) {
  typedef O vt __attribute__((ext_vector_type(8), aligned(sizeof(O))));
  const vt o = *(const vt*)p;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)o[e];
}
// the bias of columns j..j+7 (zeros without one): a lane keeps its columns from row to row
template <typename T> __device__ __forceinline__ void la_bias8(const GemmParams& p, int j, float* t) {
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = 0.f;
  if (!p.bias) return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (j + e < p.n) t[e] = p.bias_f32 ? ((const float*)p.bias)[j + e] : (float)((const T*)p.bias)[j + e];
}
template <typename T> __device__ __forceinline__ void la_finish1(const GemmParams& p, int i, int j, float x, float bias) {
  typedef typename SlopeT<T>::type S;
  const int64_t o = (int64_t)i * p.n + j;
  float s = 1.f;
  x += bias;
  la_act<T, 1>(&x, p.act, &s);
  if (p.slope) ((S*)p.slope)[o] = (S)(s * SlopeT<T>::ONE);
  if (p.res) x += (float)((const T*)p.res)[(int64_t)i * p.ldres + j];
  if (p.c_f32) ((float*)p.c)[o] = x; else ((T*)p.c)[o] = (T)x;
}
// Residuals are asked for ahead of the stores of other rows: loads and stores come back in the order of their issue, so a load
// behind a store waits for it (16384 x 1024 x 4096 bf16, GELU, slopes and a residual: 227 us, 197 so).
template <typename T> using Res8 = T __attribute__((ext_vector_type(8)));
template <typename T> __device__ __forceinline__ void la_ask8(const GemmParams& p, int i, int j, Res8<T>& t) {
  typedef T vt __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  if (p.res && i < p.m && j + 8 <= p.n) t = *(const vt*)((const T*)p.res + (int64_t)i * p.ldres + j);
}
// without an activation
template <typename T> __device__ __forceinline__ void la_plain8(const GemmParams& p, int i, int j, float* v, const float* bias, const Res8<T>& res) {
  const int64_t o = (int64_t)i * p.n + j;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += bias[e];
  if (j + 8 <= p.n) {
    if (p.res) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += (float)res[e];
    }
    if (p.c_f32) put8((float*)p.c + o, v); else put8((T*)p.c + o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e < p.n) {
        const float x = v[e] + (p.res ? (float)((const T*)p.res)[(int64_t)i * p.ldres + j + e] : 0.f);
        if (p.c_f32) ((float*)p.c)[o + e] = x; else ((T*)p.c)[o + e] = (T)x;
      }
  }
}
template <typename T> __device__ __forceinline__ void la_finish8(const GemmParams& p, int i, int j, float* v, const float* bias, const Res8<T>& res) {
  typedef typename SlopeT<T>::type S;
  const int64_t o = (int64_t)i * p.n + j;
  if (j + 8 <= p.n) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias[e];
    if (p.act != VG_ACT_NONE) {
      la_act<T, 8>(v, p.act, s);
      if (p.slope) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] *= SlopeT<T>::ONE;
        put8((S*)p.slope + o, s);
      }
    }
    if (p.res) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += (float)res[e];
    }
    if (p.c_f32) put8((float*)p.c + o, v); else put8((T*)p.c + o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e < p.n) la_finish1<T>(p, i, j + e, v[e], bias[e]);
  }
}

// ---- tiles -------------------------------------------------------------------------------------------------------------
// LDS-DMA through a buffer resource (16 bytes a lane; a lane whose offset is out of range gets zeros).  In asm, so that the
// compiler does not wait for it before LDS reads: the ring below orders them with counted waits and barriers.  M0 is put back.
typedef int la_srd_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ la_srd_t la_srd(const void* base) {
  const unsigned long long b = (unsigned long long)base;
  la_srd_t r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)(b & 0xFFFFFFFFull));
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)((b >> 32) & 0xFFFFull));
  r[2] = (int)0x80000000u;      // 2 GB of records: larger offsets are out of range
  r[3] = 0x00020000;
  return r;
}
__device__ __forceinline__ void la_dma16(la_srd_t srd, unsigned voff, unsigned lds_byte_off) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds_byte_off), "v"(voff), "s"(srd) : "memory");
}
__device__ __forceinline__ unsigned la_lds_addr(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)p;
}
template <int N> __device__ __forceinline__ void la_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
typedef __attribute__((address_space(3))) bf16x4* la_tr_t;

// One operand's tile: R rows (of C) x 128 bytes of k, in 16-byte pieces, stored so that the fragment reads below
// touch every LDS bank once.
//   k contiguous:   [row][8 pieces], piece p of row r in slot p ^ (r >> 1 & 7)
//   row contiguous: [k][R elements]; the 32-byte (f32: 64-byte) column groups of k exchanged by the bits of k in which the
//                   lanes of one read differ
constexpr int KB = 128;                              // bytes of k in a tile
template <typename T, bool TR, int R, int NTH> struct LaTile {
  static constexpr int EB = sizeof(T), PIECE = 16 / EB, KT = KB / EB, LOADS = R * (KB / 16) / NTH, BYTES = R * KB, RB = R * EB;
  static __device__ __forceinline__ int turn(int r) { return (r >> 1) & 7; }
  static constexpr int FRAG_READS = TR ? (EB == 2 ? 2 : 4) : 1;
  unsigned voff[LOADS];
  int kof[LOADS];
  __device__ __forceinline__ void init(int tid, int row0, int rows, int64_t ld) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = i * NTH + tid;
      if constexpr (!TR) {
        const int r = q / (KB / 16), pc = (q % (KB / 16)) ^ turn(r);
        kof[i] = pc * PIECE;
        voff[i] = row0 + r < rows ? (unsigned)(r * ld * EB) + pc * 16 : 0xFFFFFFFFu;
      } else {
        constexpr int PPR = RB / 16;
        const int k = q / PPR, sl = q % PPR;
        const int pc = EB == 2 ? ((((sl >> 1) ^ swz(k)) << 1) | (sl & 1)) : ((((sl >> 2) ^ swz(k)) << 2) | (sl & 3));
        kof[i] = k;
        voff[i] = row0 + pc * PIECE < rows ? (unsigned)(k * ld * EB) + pc * 16 : 0xFFFFFFFFu;
      }
    }
  }
  static __device__ __forceinline__ int swz(int k) {
    if (EB == 4) return (k >> 2) & 3;
    return RB == 128 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k & 3) | ((k >> 3) & 1) << 2;      // a 128-byte row is half the banks
  }
  // k0: first k of the tile; klimit: pieces at or beyond it come as zeros
  __device__ __forceinline__ void load(int i, la_srd_t srd, unsigned lds, int wave, int k0, int klimit) const {
    la_dma16(srd, k0 + kof[i] < klimit ? voff[i] : 0xFFFFFFFFu, lds + (i * NTH + wave * 64) * 16);
  }
  static __device__ __forceinline__ int64_t step(int64_t ld) { return TR ? KT * ld * EB : KB; }
  static __device__ __forceinline__ u32x4 frag(const unsigned char* s, int tile, int ks, int lane) {
    const int l16 = lane & 15, kg = lane >> 4;
    if constexpr (!TR) {
      const int r = tile * 16 + l16;
      return *(const u32x4*)(s + r * KB + (((ks * 4 + kg) ^ turn(r)) << 4));
    } else if constexpr (EB == 2) {
      const int tq = l16 >> 2, tp = l16 & 3, k = ks * 32 + kg * 8 + tq;
      const unsigned char* a = s + k * RB + ((tile ^ swz(k)) << 5) + tp * 8;
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_tr_t)a);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_tr_t)(a + 4 * RB));
      return __builtin_bit_cast(u32x4, bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    } else {
      const unsigned* a = (const unsigned*)(s + (ks * 16 + kg * 4) * RB + ((tile ^ kg) << 6)) + l16;
      return u32x4{a[0], a[RB / 4], a[2 * (RB / 4)], a[3 * (RB / 4)]};
    }
  }
};

__device__ __forceinline__ int la_xcd(int bid, int nblk) {      // blocks of one XCD (bid % 8) get one contiguous range of tiles
  const int q = nblk >> 3, r = nblk & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}

// WM x WN waves, each MT x NT products of 16 x 16; a ring of S tiles of k; one barrier a tile
template <typename T, bool TA, bool TB, int WM, int WN, int MT, int NT, int S>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_tile_kernel(const GemmParams p) {
  constexpr int NTH = 64 * WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
  typedef LaTile<T, TA, BM, NTH> TileA;
  typedef LaTile<T, TB, BN, NTH> TileB;
  constexpr int STAGE = TileA::BYTES + TileB::BYTES, LOADS = TileA::LOADS + TileB::LOADS, KT = TileA::KT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN, tiles = tm * tn;
  int id = la_xcd(blockIdx.x, gridDim.x);
  const int split = id / tiles;
  id -= split * tiles;
  // tiles in groups of 8 rows of tiles, so that the tiles an XCD works on at one time share rows and columns
  const int group = id / (8 * tn), gm = tm - group * 8 < 8 ? tm - group * 8 : 8;
  const int in = id - group * 8 * tn;
  const int i0 = (group * 8 + in % gm) * BM, j0 = in / gm * BN;

  TileA ta;
  TileB tb;
  ta.init(tid, i0, p.m, p.lda);
  tb.init(tid, j0, p.n, p.ldb);
  const int kt0 = split * p.ktiles, kt1 = min(kt0 + p.ktiles, (p.k + KT - 1) / KT);
  const char* ga = (const char*)p.a + (TA ? (int64_t)i0 * sizeof(T) : (int64_t)i0 * p.lda * (int64_t)sizeof(T)) + kt0 * TileA::step(p.lda);
  const char* gb = (const char*)p.b + (TB ? (int64_t)j0 * sizeof(T) : (int64_t)j0 * p.ldb * (int64_t)sizeof(T)) + kt0 * TileB::step(p.ldb);
  const int klimit = min(p.k, kt1 * KT);
  const unsigned lds0 = la_lds_addr(smem);
  int kload = kt0 * KT, slot = 0;
  la_srd_t srd_a, srd_b;
  unsigned base;
  auto begin = [&]() { srd_a = la_srd(ga); srd_b = la_srd(gb); base = lds0 + slot * STAGE; };
  auto load = [&](int i) {
    if (i < TileA::LOADS) ta.load(i, srd_a, base, wave, kload, klimit);
    else tb.load(i - TileA::LOADS, srd_b, base + TileA::BYTES, wave, kload, klimit);
  };
  auto end = [&]() {
    if (kload + KT < klimit) { ga += TileA::step(p.lda); gb += TileB::step(p.ldb); }      // past the end only zeros are asked for
    kload += KT;
    slot = slot + 1 == S ? 0 : slot + 1;
  };
  f32x4 acc[MT][NT] = {};
  // Two sets of fragments: while the products of one half of a tile run, the other half (or the next tile's first half) is
  // read from LDS and the tile after the next is asked for, a few of each between the rows of products.  All reads first and
  // all products after leaves each unit idle half of the time (8192 x 4096 x 4096: 248 us).
  u32x4 fa[2][MT], fb[2][NT];
  auto read = [&](int set, const unsigned char* s, int ks, int i) {      // the columns' fragments first: every row needs them
    if (i < NT) fb[set][i] = TileB::frag(s + TileA::BYTES, wn * NT + i, ks, lane);
    else fa[set][i - NT] = TileA::frag(s, wm * MT + i - NT, ks, lane);
  };
  constexpr int FRAGS = MT + NT, PER = (FRAGS + MT - 2) / (MT - 1), DMA = (LOADS + MT - 1) / MT;
  auto multiply = [&](int set, const unsigned char* s, int ks, bool ask) {
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      if (ask) {
#pragma unroll
        for (int i = u * DMA; i < (u + 1) * DMA && i < LOADS; ++i) load(i);
      }
#pragma unroll
      for (int i = u * PER; i < (u + 1) * PER && i < FRAGS; ++i) read(set ^ 1, s, ks, i);
#pragma unroll
      for (int v = 0; v < NT; ++v) acc[u][v] = la_mma<T>(fb[set][v], fa[set][u], acc[u][v]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
    begin();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(i);
    end();
  }
  la_wait_barrier<(S - 1) * LOADS>();
#pragma unroll
  for (int i = 0; i < FRAGS; ++i) read(0, smem, 0, i);
  int cur = 0;
  for (int kt = kt0; kt < kt1; ++kt) {
    multiply(0, smem + cur * STAGE, 1, false);
    la_wait_barrier<(S - 2) * LOADS>();              // the next tile is in LDS, and everyone has read this one
    cur = cur + 1 == S ? 0 : cur + 1;
    begin();                                         // tile kt + S takes its place; past the last one: zeros
    multiply(1, smem + cur * STAGE, 0, true);
    end();
  }
  la_wait_barrier<0>();                              // the zeros asked for past the end have landed: LDS is free

  // acc[u][v][r] of a lane: row 16 u + lane % 16, column 16 v + 4 (lane / 16) + r.
  constexpr bool WIDE = sizeof(T) == 4 || NT == 2;   // the four lanes of a row read all that the wave has of it, or a line
  if (p.part || (p.act == VG_ACT_NONE && (WIDE || !p.res))) {
    // Two neighbouring 16 x 16 blocks exchange rows of lanes, after which a lane has eight neighbouring columns: of the left
    // block in lanes 0-15 and 32-47, of the right one in the others.
    const int i1 = i0 + wm * MT * 16 + (lane & 15), j1 = j0 + wn * NT * 16 + ((lane >> 4) & 1) * 16 + (lane >> 5) * 8;
    Res8<T> res[NT / 2][MT];
    if (WIDE && !p.part && p.res) {
#pragma unroll
      for (int v = 0; v < NT; v += 2)
#pragma unroll
        for (int u = 0; u < MT; ++u) la_ask8<T>(p, i1 + u * 16, j1 + v * 16, res[v / 2][u]);
    }
#pragma unroll
    for (int v = 0; v < NT; v += 2) {
      const int j = j1 + v * 16;
      float bias[8];
      if (!p.part) la_bias8<T>(p, j, bias);
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[u][v][r]), __float_as_uint(acc[u][v + 1][r]), false, false);
          x[r] = __uint_as_float(s[0]);
          x[4 + r] = __uint_as_float(s[1]);
        }
        const int i = i1 + u * 16;
        if (i < p.m && j < p.n) {
          if (p.part) put8(p.part + ((int64_t)split * p.m + i) * p.ldp + j, x);
          else la_plain8<T>(p, i, j, x, bias, res[v / 2][u]);
        }
      }
    }
    return;
  }
  // Through LDS (half of the wave's rows at a time) into a loop: with an activation, since sixteen copies of it would not stay in
  // the instruction cache; bf16 residuals, since the eight lanes of a row read whole lines (16384 x 1024 x 4096 without an
  // activation: 170 us by halves of lines, 149 so).
  constexpr int LDW = 16 * NT + 4, HALF = MT / 2;
  static_assert(64 % (2 * NT) == 0, "a lane keeps its columns");
  float* st = (float*)smem + wave * 16 * HALF * LDW;
  const int c = (lane % (2 * NT)) * 8, j = j0 + wn * NT * 16 + c;
  constexpr int ITER = NT * HALF / 2, BATCH = ITER < 4 ? ITER : 4;      // accesses of a lane to a half; how many residuals wait
  const int iw = i0 + wm * MT * 16;
  float bias[8];
  la_bias8<T>(p, j, bias);
  Res8<T> res[BATCH], next[BATCH];
  auto ask = [&](int q) {                            // the q-th access of a lane is to row (q * 64 + lane) / (2 NT) of the wave's
#pragma unroll
    for (int b = 0; b < BATCH; ++b) la_ask8<T>(p, iw + ((q + b) * 64 + lane) / (2 * NT), j, next[b]);
  };
  ask(0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int u = 0; u < HALF; ++u)
#pragma unroll
      for (int v = 0; v < NT; ++v) *(f32x4*)(st + (u * 16 + (lane & 15)) * LDW + v * 16 + (lane >> 4) * 4) = acc[h * HALF + u][v];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
    for (int t0 = 0; t0 < ITER; t0 += BATCH) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b) res[b] = next[b];
      if (h * ITER + t0 + BATCH < 2 * ITER) ask(h * ITER + t0 + BATCH);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int r = ((t0 + b) * 64 + lane) / (2 * NT), i = iw + h * HALF * 16 + r;
        float v[8];
        *(f32x4*)v = *(const f32x4*)(st + r * LDW + c);
        *(f32x4*)(v + 4) = *(const f32x4*)(st + r * LDW + c + 4);
        if (i < p.m && j < p.n) la_finish8<T>(p, i, j, v, bias, res[b]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// ---- few rows (m <= 64): one read of the weights -------------------------------------------------------------------------
// A block takes 16 columns of C; its eight waves take k by turns of 4 x 64 bytes and join their sums in LDS, so the weights
// stream from memory with 4 KB of each wave in flight and there is no second launch.  TW: f32 master weights are rounded here.
// WHOLE: k is a whole number of pieces.
template <typename T, typename TW, bool WHOLE> __device__ __forceinline__ u32x4 la_piece(const TW* row, int64_t k, int64_t kmax) {
  constexpr int P = 16 / sizeof(T);
  typedef T vt __attribute__((ext_vector_type(P)));
  vt v;
  if (WHOLE ? k >= kmax : k + P > kmax) {
    if constexpr (WHOLE) return u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] = k + e < kmax ? (T)(float)row[k + e] : (T)0.f;
  } else {
    typedef TW wt __attribute__((ext_vector_type(P), aligned(sizeof(TW))));
    const wt q = *(const wt*)(row + k);
    if constexpr (sizeof(TW) == sizeof(T)) return __builtin_bit_cast(u32x4, q);
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] = (T)q[e];
  }
  return __builtin_bit_cast(u32x4, v);
}
template <typename T, typename TW, int MB, bool WHOLE>
__global__ __launch_bounds__(512) void gemm_rows_kernel(const GemmParams p) {
  constexpr int P = 16 / sizeof(T), STEP = 4 * P, U = 4;        // k of one matrix instruction group, and how many a turn
  __shared__ float part[8][MB * 16][16 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, kg = lane >> 4;
  const int j0 = blockIdx.x * 16;
  const T* A = (const T*)p.a;
  const TW* B = (const TW*)p.b + (int64_t)min(j0 + l16, p.n - 1) * p.ldb;       // columns past n repeat the last one and are not stored
  const T* rows[MB];
#pragma unroll
  for (int u = 0; u < MB; ++u) rows[u] = A + (int64_t)min(u * 16 + l16, p.m - 1) * p.lda;
  f32x4 acc[MB] = {};
  for (int64_t k0 = (int64_t)wave * U * STEP; k0 < p.k; k0 += 8 * U * STEP) {
    u32x4 w[U], x[U][MB];
#pragma unroll
    for (int t = 0; t < U; ++t) w[t] = la_piece<T, TW, WHOLE>(B, k0 + t * STEP + kg * P, p.k);
#pragma unroll
    for (int t = 0; t < U; ++t)
#pragma unroll
      for (int u = 0; u < MB; ++u) x[t][u] = la_piece<T, T, WHOLE>(rows[u], k0 + t * STEP + kg * P, p.k);
#pragma unroll
    for (int t = 0; t < U; ++t)
#pragma unroll
      for (int u = 0; u < MB; ++u) acc[u] = la_mma<T>(w[t], x[t][u], acc[u]);
  }
  // acc[u][r]: row 16 u + lane % 16 of C, column 4 (lane / 16) + r
#pragma unroll
  for (int u = 0; u < MB; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][u * 16 + l16][kg * 4 + r] = acc[u][r];
  __syncthreads();
  for (int q = threadIdx.x; q < MB * 256; q += 512) {
    const int i = q >> 4, c = q & 15, j = j0 + c;
    if (i >= p.m || j >= p.n) continue;
    float v = part[0][i][c];
#pragma unroll
    for (int s = 1; s < 8; ++s) v += part[s][i][c];
    const float bias = p.bias ? p.bias_f32 ? ((const float*)p.bias)[j] : (float)((const T*)p.bias)[j] : 0.f;
    la_finish1<T>(p, i, j, v, bias);
  }
}

// sums of the splits in their order, and the epilogue
template <typename T> __global__ __launch_bounds__(256) void gemm_join_kernel(const GemmParams p) {
  const int per = p.ldp / 8;
  const int64_t q = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (q >= (int64_t)p.m * per) return;
  const int i = (int)(q / per), j = (int)(q % per) * 8;
  float v[8], t[8];
  Res8<T> res;
  la_ask8<T>(p, i, j, res);
  get8(p.part + (int64_t)i * p.ldp + j, v);
  for (int s = 1; s < p.splits; ++s) {
    get8(p.part + ((int64_t)s * p.m + i) * p.ldp + j, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  float bias[8];
  la_bias8<T>(p, j, bias);
  la_finish8<T>(p, i, j, v, bias, res);
}

// Matrices [rows][cols] (row stride ld) into [rows][pitch], the padding zeroed: both operands of a product in one launch, the
// first taking `split` blocks.  f32 sources of bf16 products (master weights) are rounded.
struct PackParams {
  const void* src[2];
  void* dst[2];
  int64_t ld[2], rows[2];
  int cols[2], pitch[2], f32[2];
  unsigned split;
};
template <typename S, typename T>
__device__ __forceinline__ void la_pack_one(const S* src, int64_t ld, T* dst, int64_t rows, int cols, int pitch, int64_t block, int64_t blocks) {
  const int per = pitch / 8;
  for (int64_t q = block * 256 + threadIdx.x; q < rows * per; q += blocks * 256) {
    const int64_t r = q / per;
    const int c = (int)(q % per) * 8;
    float v[8];
    if (c + 8 <= cols) get8(src + r * ld + c, v);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? (float)src[r * ld + c + e] : 0.f;
    }
    put8(dst + r * pitch + c, v);
  }
}
template <typename T> __global__ __launch_bounds__(256) void la_pack_kernel(const PackParams p) {
  const int w = blockIdx.x >= p.split;
  const int64_t block = w ? blockIdx.x - p.split : blockIdx.x, blocks = w ? gridDim.x - p.split : p.split;
  if (sizeof(T) == 2 && p.f32[w]) la_pack_one((const float*)p.src[w], p.ld[w], (T*)p.dst[w], p.rows[w], p.cols[w], p.pitch[w], block, blocks);
  else la_pack_one((const T*)p.src[w], p.ld[w], (T*)p.dst[w], p.rows[w], p.cols[w], p.pitch[w], block, blocks);
}

// dz = dy slope (dz = dy without one) and partial column sums of the unrounded dz: part[row chunk][n].
// A block is 32 column groups of 8 (512 bytes of a row) by 8 rows, so 16-byte accesses and runs of memory; bound by one read
// of dy and slope and one write of dz.  The backward pass reads neither of the two again (dy may be, as the residual's gradient),
// so they do not take the cache from dz, which both products read next (bf16 16384 x 1024 x 4096, forward + backward: 528 us with
// ordinary loads, 500 so).
template <typename T>
__global__ __launch_bounds__(256) void la_dz_kernel(const T* __restrict__ dy, const typename SlopeT<T>::type* __restrict__ slope, T* __restrict__ dz,
                                                    float* __restrict__ part, int m, int n, int rows_per) {
  __shared__ float fold[8][257];
  const int cg = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int j = (blockIdx.x * 32 + cg) * 8;
  const int r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < m ? r0 + rows_per : m;
  float s[8] = {};
  auto rows = [&](auto whole) {                      // the last columns of a row that is no multiple of 8: element by element
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll 4
    for (int r = r0 + ry; r < r1; r += 8) {
      const int64_t o = (int64_t)r * n + j;
      float g[8], t[8];
      if constexpr (WHOLE) { if (slope) get8_nt(dy + o, g); else get8(dy + o, g); }
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = j + e < n ? (float)dy[o + e] : 0.f;
      }
      if (slope) {
        if constexpr (WHOLE) get8_nt(slope + o, t);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = j + e < n ? (float)slope[o + e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= t[e] * (1.f / SlopeT<T>::ONE);
        if constexpr (WHOLE) put8(dz + o, g);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (j + e < n) dz[o + e] = (T)g[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += g[e];
    }
  };
  if (j + 8 <= n) rows(std::true_type{});
  else if (j < n) rows(std::false_type{});
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) fold[ry][cg * 8 + e] = s[e];
  __syncthreads();
  const int c = threadIdx.x, col = blockIdx.x * 256 + c;
  float t = fold[0][c];
#pragma unroll
  for (int q = 1; q < 8; ++q) t += fold[q][c];
  if (col < n) part[(int64_t)blockIdx.y * n + col] = t;
}

// ---- host --------------------------------------------------------------------------------------------------------------
// An operand as the tiles read it: the caller's matrix where it has 16-byte rows, otherwise a zero-padded copy.
struct LaOperand {
  const void* p;
  int64_t ld, rows, cols;       // of the stored matrix
  int src_f32;                  // f32 master weight of bf16 products
};
static size_t la_up(size_t n) { return (n + 255) / 256 * 256; }
static int64_t la_pitch(int64_t cols) { return (cols + 7) / 8 * 8; }
static bool la_direct(const LaOperand& o, int dtype) {
  const int e = vg_elt_size(dtype);
  return !(o.src_f32 && dtype == VG_BF16) && (uintptr_t)o.p % 16 == 0 && o.cols % (16 / e) == 0 && (o.ld * e) % 16 == 0 && o.ld * e < (1LL << 23);      // 255 rows within 2 GB
}
static size_t la_packed_bytes(const LaOperand& o, int dtype) { return la_up((size_t)o.rows * la_pitch(o.cols) * vg_elt_size(dtype)); }

// Which tiles, and how many ways the contraction is split (partial sums in f32, joined by a kernel): the cheapest by an estimate
// from measured times (us).  A CU with nb blocks takes max(lat, nb * step) for 128 bytes of k of each, and `fixed` for the ends
// of every `res` blocks that it holds at once; a join costs its launch and the partial sums' way out and back.
//   tile    bf16 lat  step  fixed  res     f32 lat  step  fixed
//   64          0.26  0.20   2.5    3         0.6   0.53   3.0
//   128         0.68  0.55   3.5    2         2.0   2.0    5.0
//   256         1.50  1.65   6.0    1
// E.g. bf16 1024^3: 64 unsplit 6.9, 128 unsplit 12.1, 128 in eight 25; dW of 16384 x 1024 x 4096: 256 in four 145, 128 in two 187;
// forward of 16381 x 2048 x 512: 128 39, 256 57.
struct LaPlan { int tile, splits, ktiles; double us; };
static LaPlan la_plan(int64_t m, int64_t n, int64_t k, int dtype) {
  struct Cost { int tile, res; double lat, step, fixed; };
  static const Cost bf16[3] = {{64, 3, 0.26, 0.20, 2.5}, {128, 2, 0.68, 0.55, 3.5}, {256, 1, 1.50, 1.65, 6.0}};
  static const Cost f32[2] = {{64, 3, 0.6, 0.53, 3.0}, {128, 2, 2.0, 2.0, 5.0}};
  const int64_t kt = vg_ceil_div(k * vg_elt_size(dtype), KB);
  LaPlan best = {64, 1, (int)kt, 1e30};
  for (int i = 0; i < (dtype == VG_BF16 ? 3 : 2); ++i) {
    const Cost& c = dtype == VG_BF16 ? bf16[i] : f32[i];
    const int64_t tiles = vg_ceil_div(m, c.tile) * vg_ceil_div(n, c.tile);
    for (int64_t s = 1; s <= 32 && (s == 1 || kt / s >= 4); s += s < 4 ? 1 : s < 8 ? 2 : 4) {
      const int64_t per = vg_ceil_div(kt, s), parts = vg_ceil_div(kt, per), nb = vg_ceil_div(tiles * parts, 256);
      const double join = parts > 1 ? 4.5 + (double)parts * m * n * 1.07e-6 : 0;
      const double us = per * (nb * c.step > c.lat ? nb * c.step : c.lat) + c.fixed * vg_ceil_div(nb, c.res) + join;
      if (us < best.us) best = {c.tile, (int)parts, (int)per, us};
    }
  }
  return best;
}
static size_t la_part_bytes(int64_t m, int64_t n, int64_t k, int dtype) {
  const LaPlan pl = la_plan(m, n, k, dtype);
  return pl.splits > 1 ? la_up((size_t)pl.splits * m * la_pitch(n) * sizeof(float)) : 0;
}
static size_t la_ws(int64_t m, int64_t n, int64_t k, int dtype, const LaOperand& a, const LaOperand& b) {
  return la_part_bytes(m, n, k, dtype) + (la_direct(a, dtype) ? 0 : la_packed_bytes(a, dtype)) + (la_direct(b, dtype) ? 0 : la_packed_bytes(b, dtype));
}

// copies what the tiles cannot read in place to the workspace; returns its first free byte
static char* la_pack(LaOperand* o[2], int dtype, char* ws, hipStream_t st) {
  PackParams p = {};
  unsigned blocks[2] = {0, 0};
  int n = 0;
  for (int i = 0; i < 2; ++i) {
    if (la_direct(*o[i], dtype)) continue;
    const int64_t pitch = la_pitch(o[i]->cols), need = vg_ceil_div(o[i]->rows * (pitch / 8), 256);
    p.src[n] = o[i]->p; p.dst[n] = ws; p.ld[n] = o[i]->ld; p.rows[n] = o[i]->rows; p.cols[n] = (int)o[i]->cols; p.pitch[n] = (int)pitch; p.f32[n] = o[i]->src_f32;
    blocks[n++] = (unsigned)(need < 8192 ? need : 8192);
    const size_t bytes = la_packed_bytes(*o[i], dtype);
    o[i]->p = ws; o[i]->ld = pitch;
    ws += bytes;
  }
  if (n) {
    p.split = blocks[0];
    if (dtype == VG_BF16) hipLaunchKernelGGL(la_pack_kernel<bf16_t>, dim3(blocks[0] + blocks[1]), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(la_pack_kernel<float>, dim3(blocks[0] + blocks[1]), dim3(256), 0, st, p);
  }
  return ws;
}

// what the calling thread's last product ran on (vg_last_linear_act_kernel)
static thread_local struct { int rows, tile, ta, tb, splits, f32; } la_last;
extern "C" const char* vg_last_linear_act_kernel(void) {
  static thread_local char name[64];
  if (la_last.rows) snprintf(name, sizeof(name), "rows<%s,%d>", la_last.f32 ? "f32" : "bf16", la_last.rows);
  else snprintf(name, sizeof(name), "tile<%s,%d,%c%c>%s", la_last.f32 ? "f32" : "bf16", la_last.tile, la_last.ta ? 't' : 'n', la_last.tb ? 't' : 'n', la_last.splits > 1 ? "+join" : "");
  return name;
}

template <typename T, bool TA, bool TB, int WM, int WN, int MT, int NT, int S> static int la_tile_launch(GemmParams p, hipStream_t st) {
  constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN;
  const int ring = S * (BM + BN) * KB, out = WM * WN * 8 * MT * (16 * NT + 4) * 4, lds = ring > out ? ring : out;
  void (*kernel)(const GemmParams) = gemm_tile_kernel<T, TA, TB, WM, WN, MT, NT, S>;
  VG_HIP(vg_lds_attr((const void*)kernel, lds));
  const int64_t blocks = vg_ceil_div(p.m, BM) * vg_ceil_div(p.n, BN) * p.splits;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WM * WN), lds, st, p);
  VG_LAUNCH_CHECK();
  return VG_OK;
}
template <typename T, bool TA, bool TB> static int la_gemm_t(GemmParams p, const LaPlan& pl, int dtype, char* ws, hipStream_t st) {
  p.splits = pl.splits;
  p.ktiles = pl.ktiles;
  p.ldp = (int)la_pitch(p.n);
  p.part = pl.splits > 1 ? (float*)ws : nullptr;
  la_last = {0, pl.tile, TA, TB, pl.splits, dtype == VG_F32};
  int rc;
  if (pl.tile == 64) rc = la_tile_launch<T, TA, TB, 2, 2, 2, 2, 3>(p, st);
  else if (pl.tile == 128) rc = la_tile_launch<T, TA, TB, 2, 2, 4, 4, 2>(p, st);
  else {
    if constexpr (sizeof(T) == 2) rc = la_tile_launch<T, TA, TB, 2, 4, 8, 4, 2>(p, st);
    else rc = VG_ERR_UNSUPPORTED;                    // not planned for f32, whose matrix rate binds at any size
  }
  if (rc) return rc;
  if (pl.splits > 1) {
    hipLaunchKernelGGL(gemm_join_kernel<T>, dim3((unsigned)vg_ceil_div((int64_t)p.m * (p.ldp / 8), 256)), dim3(256), 0, st, p);
    VG_LAUNCH_CHECK();
  }
  return VG_OK;
}
// C [m][n] = A B over k; a is stored [m][k] (ta: [k][m]), b [n][k] (tb: [k][n])
static int la_gemm(GemmParams p, LaOperand a, bool ta, LaOperand b, bool tb, int dtype, void* ws, hipStream_t st) {
  VG_REQUIRE((uintptr_t)ws % 256 == 0 && (ws || la_ws(p.m, p.n, p.k, dtype, a, b) == 0), "linear_act: needs a workspace, aligned to 256 bytes");
  const LaPlan pl = la_plan(p.m, p.n, p.k, dtype);
  VG_GRID_CHECK("linear_act", vg_ceil_div(p.m, pl.tile) * vg_ceil_div(p.n, pl.tile) * pl.splits, pl.tile == 256 ? 512 : 256);
  LaOperand* both[2] = {&a, &b};
  char* w = la_pack(both, dtype, (char*)ws, st);
  p.a = a.p; p.lda = a.ld; p.b = b.p; p.ldb = b.ld;
  if (dtype == VG_BF16)
    return ta ? la_gemm_t<bf16_t, true, true>(p, pl, dtype, w, st) : tb ? la_gemm_t<bf16_t, false, true>(p, pl, dtype, w, st) : la_gemm_t<bf16_t, false, false>(p, pl, dtype, w, st);
  return ta ? la_gemm_t<float, true, true>(p, pl, dtype, w, st) : tb ? la_gemm_t<float, false, true>(p, pl, dtype, w, st) : la_gemm_t<float, false, false>(p, pl, dtype, w, st);
}

// Whether the few-rows kernel takes a forward product: its time is bound by one read of the weights from memory (3.9 TB/s) or
// by every block's read of x from the cache (7 TB/s), against the tiles' and the copies that they need of f32 master weights
// or of rows that are not whole 16-byte pieces.  bf16 64 x 1024 x 4096: 8.0 us here, 6.7 in tiles; 32 rows: 5.7 and 6.7; 64
// rows with f32 weights: 9.1 and 25.
static bool la_few_rows(int64_t m, int64_t n, int64_t k, int dtype, const LaOperand& x, const LaOperand& w) {
  if (m > 64) return false;
  const double e = vg_elt_size(dtype), ew = w.src_f32 ? 4 : e;
  const double read = n * (double)k * ew / 3.9e6, cached = vg_ceil_div(n, 16) * (double)m * k * e / 7e6;
  const double few = 2.5 + (read > cached ? read : cached);
  double tiles = la_plan(m, n, k, dtype).us;
  if (!la_direct(w, dtype)) tiles += 3 + n * (double)k * (ew + e) / 4e6;
  if (!la_direct(x, dtype)) tiles += 3;
  return few <= tiles;
}
template <typename T, typename TW, int MB> static void la_rows_launch(const GemmParams& p, bool whole, hipStream_t st) {
  const dim3 grid((unsigned)vg_ceil_div(p.n, 16));
  if (whole) hipLaunchKernelGGL((gemm_rows_kernel<T, TW, MB, true>), grid, dim3(512), 0, st, p);
  else hipLaunchKernelGGL((gemm_rows_kernel<T, TW, MB, false>), grid, dim3(512), 0, st, p);
}
template <typename T, typename TW> static int la_rows(const GemmParams& p, hipStream_t st) {
  la_last = {p.m <= 16 ? 16 : p.m <= 32 ? 32 : 64, 0, 0, 0, 1, sizeof(T) == 4};
  const bool whole = p.k % (16 / sizeof(T)) == 0;
  if (p.m <= 16) la_rows_launch<T, TW, 1>(p, whole, st);
  else if (p.m <= 32) la_rows_launch<T, TW, 2>(p, whole, st);
  else la_rows_launch<T, TW, 4>(p, whole, st);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

static int la_check(const char* what, int64_t m, int64_t n, int64_t k, int act, int dtype) {
  VG_REQUIRE(dtype == VG_F32 || dtype == VG_BF16, "%s: dtype %d", what, dtype);
  VG_REQUIRE(m >= 1 && n >= 1 && k >= 1 && m < (1LL << 30) && n < (1LL << 20) && k < (1LL << 20), "%s: %ld x %ld x %ld", what, (long)m, (long)n, (long)k);
  VG_REQUIRE(act >= VG_ACT_NONE && act <= VG_ACT_SILU, "%s: activation %d", what, act);
  return VG_OK;
}
static int la_weight(const char* what, int w_dtype, int dtype) {
  VG_REQUIRE(w_dtype == dtype || w_dtype == VG_F32, "%s: weight dtype %d for dtype %d", what, w_dtype, dtype);
  return VG_OK;
}

extern "C" size_t vg_linear_act_fwd_ws_bytes(const void* x, int64_t ldx, const void* w, int w_dtype, int64_t m, int64_t n, int64_t k, int dtype) {
  const LaOperand a = {x, ldx, m, k, 0}, b = {w, k, n, k, w_dtype == VG_F32};
  return la_few_rows(m, n, k, dtype, a, b) ? 0 : la_ws(m, n, k, dtype, a, b);
}
extern "C" int vg_linear_act_fwd(const void* x, int64_t ldx, const void* w, int w_dtype, const void* bias, int bias_dtype, const void* res,
                                 int64_t ldres, void* y, void* slope, void* ws, int64_t m, int64_t n, int64_t k, int act, int dtype,
                                 void* stream) {
  if (int rc = la_check("linear_act_fwd", m, n, k, act, dtype)) return rc;
  if (int rc = la_weight("linear_act_fwd", w_dtype, dtype)) return rc;
  VG_REQUIRE(x && w && y && ldx >= k && (!res || ldres >= n), "linear_act_fwd: null pointer or a short row stride");
  GemmParams p = {};
  p.m = (int)m; p.n = (int)n; p.k = (int)k;
  p.c = y; p.bias = bias; p.bias_f32 = bias_dtype == VG_F32; p.res = res; p.ldres = ldres; p.slope = act == VG_ACT_NONE ? nullptr : slope; p.act = act;
  const LaOperand a = {x, ldx, m, k, 0}, b = {w, k, n, k, w_dtype == VG_F32};
  if (la_few_rows(m, n, k, dtype, a, b)) {
    p.a = x; p.lda = ldx; p.b = w; p.ldb = k;
    if (dtype == VG_F32) return la_rows<float, float>(p, (hipStream_t)stream);
    return w_dtype == VG_F32 ? la_rows<bf16_t, float>(p, (hipStream_t)stream) : la_rows<bf16_t, bf16_t>(p, (hipStream_t)stream);
  }
  return la_gemm(p, a, false, b, false, dtype, ws, (hipStream_t)stream);
}

// chunks of rows: enough blocks to fill the chip, at least 16 rows each so that the partial sums stay a small part of the traffic
static int la_dz_parts(int64_t m, int64_t n) {
  int64_t parts = vg_ceil_div(2048, vg_ceil_div(n, 256));
  if (parts > vg_ceil_div(m, 16)) parts = vg_ceil_div(m, 16);
  return (int)parts;
}
extern "C" size_t vg_linear_act_dz_ws_bytes(int64_t m, int64_t n) {
  return m < 1 || n < 1 ? 0 : (size_t)la_dz_parts(m, n) * (size_t)n * sizeof(float);
}
extern "C" int vg_linear_act_dz(const void* dy, const void* slope, void* dz, void* db, int bias_dtype, void* ws, int64_t m, int64_t n,
                                int dtype, void* stream) {
  if (int rc = la_check("linear_act_dz", m, n, 1, VG_ACT_NONE, dtype)) return rc;
  VG_REQUIRE(dy && (!slope || dz) && (slope || db) && (!db || ws), "linear_act_dz: null pointer");
  hipStream_t st = (hipStream_t)stream;
  const int per = (int)vg_ceil_div(m, la_dz_parts(m, n)), parts = (int)vg_ceil_div(m, per);
  float* part = db ? (float*)ws : nullptr;
  const dim3 grid((unsigned)vg_ceil_div(n, 256), (unsigned)parts);
  if (dtype == VG_BF16) hipLaunchKernelGGL(la_dz_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t*)dy, (const f16_t*)slope, (bf16_t*)dz, part, (int)m, (int)n, per);
  else hipLaunchKernelGGL(la_dz_kernel<float>, grid, dim3(256), 0, st, (const float*)dy, (const float*)slope, (float*)dz, part, (int)m, (int)n, per);
  VG_LAUNCH_CHECK();
  if (db) return vg_fold_cols(part, parts, n, db, n, nullptr, bias_dtype, st);
  return VG_OK;
}

extern "C" size_t vg_linear_act_dgrad_ws_bytes(const void* dz, const void* w, int w_dtype, int64_t m, int64_t n, int64_t k, int dtype) {
  return la_ws(m, k, n, dtype, {dz, n, m, n, 0}, {w, k, n, k, w_dtype == VG_F32});
}
extern "C" int vg_linear_act_dgrad(const void* dz, const void* w, int w_dtype, void* dx, void* ws, int64_t m, int64_t n, int64_t k, int dtype,
                                   void* stream) {
  if (int rc = la_check("linear_act_dgrad", m, n, k, VG_ACT_NONE, dtype)) return rc;
  if (int rc = la_weight("linear_act_dgrad", w_dtype, dtype)) return rc;
  VG_REQUIRE(dz && w && dx, "linear_act_dgrad: null pointer");
  GemmParams p = {};
  p.m = (int)m; p.n = (int)k; p.k = (int)n;
  p.c = dx;
  return la_gemm(p, {dz, n, m, n, 0}, false, {w, k, n, k, w_dtype == VG_F32}, true, dtype, ws, (hipStream_t)stream);
}

extern "C" size_t vg_linear_act_wgrad_ws_bytes(const void* dz, const void* x, int64_t ldx, int64_t m, int64_t n, int64_t k, int dtype) {
  return la_ws(n, k, m, dtype, {dz, n, m, n, 0}, {x, ldx, m, k, 0});
}
extern "C" int vg_linear_act_wgrad(const void* dz, const void* x, int64_t ldx, void* dw, int dw_dtype, void* ws, int64_t m, int64_t n, int64_t k,
                                   int dtype, void* stream) {
  if (int rc = la_check("linear_act_wgrad", m, n, k, VG_ACT_NONE, dtype)) return rc;
  if (int rc = la_weight("linear_act_wgrad", dw_dtype, dtype)) return rc;
  VG_REQUIRE(dz && x && dw && ldx >= k, "linear_act_wgrad: null pointer or a short row stride");
  GemmParams p = {};
  p.m = (int)n; p.n = (int)k; p.k = (int)m;
  p.c = dw; p.c_f32 = dw_dtype == VG_F32;
  return la_gemm(p, {dz, n, m, n, 0}, true, {x, ldx, m, k, 0}, true, dtype, ws, (hipStream_t)stream);
}

// Log probabilities of given tokens under rows of logits, with the entropy and the best alternatives, and their gradient.
//   m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m):  lse = m + ln s,  logp = x_t - lse,  H = ln s - u / s
//   dx_j = dlogp ([j = t] - p_j) - dH p_j (ln p_j + H),  p_j = e^(x_j - lse)
// Bound by memory: the forward reads the logits once, keeping (m, s, u) as running values that are rescaled when a larger
// maximum arrives; the backward reads them once more and writes the gradient.  Sums are f32; exponents are of x - m <= 0.
// Masked logits (-inf) count for nothing.  A row of nothing but -inf has no distribution: logp -inf, H 0, gradient 0.  A
// NaN or +inf in a row makes its logp, H and gradient NaN.  tokens[r] == ignore: logp 0 and no gradient through logp; any
// other token outside [0, vocab) gives logp NaN and no gradient through logp (it is never used as an index).
#include "common.h"
#include "rows.h"

#define LP_MAX_TOP 32
#define LP_CAND 512        // candidates a block can hold for the selection of the best

template <typename T> __device__ __forceinline__ float ldf(const T* p) { return (float)*p; }

// A set's maximum m, s = sum 2^d and u = sum 2^d d with d = (x - m) log2 e: one fused multiply-add and one exponential an
// element.  Masked elements have d = -inf: clamped where it multiplies, since 0 * -inf is NaN (2^-290 is 0 in f32).
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f
struct Soft { float m, s, u; };
__device__ __forceinline__ float safe_max(float m) { return m == -__builtin_inff() ? 0.f : m; }
// the same set about another maximum
__device__ __forceinline__ Soft soft_about(const Soft& a, float m) {
  const float d = fmaxf((a.m - safe_max(m)) * LP_LOG2E, -290.f), e = __builtin_amdgcn_exp2f(d);
  return Soft{m, a.s * e, e * (a.u + d * a.s)};
}
// (m, s, u) of two disjoint sets
__device__ __forceinline__ Soft soft_join(const Soft& a, const Soft& b) {
  const float m = fmaxf(a.m, b.m);
  const Soft p = soft_about(a, m), q = soft_about(b, m);
  return Soft{m, p.s + q.s, p.u + q.u};
}
__device__ __forceinline__ void soft_add(Soft& a, float x, float base) {
  const float d = (x - base) * LP_LOG2E, e = __builtin_amdgcn_exp2f(d);
  a.s += e;
  a.u += e * fmaxf(d, -290.f);
}
template <int N> __device__ __forceinline__ void soft_add_n(Soft& a, const float* x) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
  if (mx > a.m) a = soft_about(a, mx);
  const float base = safe_max(a.m);
#pragma unroll
  for (int i = 0; i < N; ++i) soft_add(a, x[i], base);
}
__device__ __forceinline__ Soft soft_wave(const Soft& a) {
  const Soft b = soft_about(a, wave_max64(a.m));
  return Soft{b.m, wave_sum64(b.s), wave_sum64(b.u)};
}

// order of the alternatives: by value, then by place (lower first); NaN ranks as -inf, -0 as +0.  A larger key is better.
__device__ __forceinline__ unsigned long long rank_key(float x, unsigned at) {
  x = x == x ? x + 0.f : -__builtin_inff();
  const unsigned b = __float_as_uint(x);
  const unsigned o = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)o << 32) | (0xFFFFFFFFu - at);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned key_place(unsigned long long k) { return 0xFFFFFFFFu - (unsigned)k; }
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long b = __shfl_xor(k, o, 64);
    k = b > k ? b : k;
  }
  return k;
}

// the `top` largest of n different keys, to put(k, key), by one wave
template <typename F> __device__ __forceinline__ void best_of(const unsigned long long* keys, int n, int top, int lane, F put) {
  if (n <= 64) {                                     // each lane counts the keys above its own
    const unsigned long long mine = lane < n ? keys[lane] : 0;
    int above = 0;
    for (int q = 0; q < n; ++q) above += keys[q] > mine;
    if (lane < n && mine && above < top) put(above, mine);
    return;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long b = 0;
    for (int q = lane; q < n; q += 64)
      if (keys[q] < last && keys[q] > b) b = keys[q];
    last = wave_max_key(b);
    if (lane == 0) put(k, last);
  }
}

struct LpParams {
  const void* x;
  int64_t ldx;
  const int64_t* tokens;
  int64_t ignore;
  int64_t rows;
  int vocab, top, splits, chunk;      // chunk: elements of a split (a multiple of 8)
  float *logp, *entropy, *lse;
  float* top_logp;
  int64_t* top_at;
  float* part;                        // [rows][splits][4]: m, s, u of a split
  unsigned long long* cand;           // [rows][splits][top]: its best
};

__device__ __forceinline__ void finish_row(const LpParams& p, int64_t row, const Soft& a, float xt) {
  const bool empty = a.m == -__builtin_inff() && a.s == 0.f;
  const float ls = logf(a.s);
  const int64_t t = p.tokens[row];
  p.entropy[row] = empty ? 0.f : ls - a.u / a.s * LP_LN2;
  p.logp[row] = t == p.ignore ? 0.f : (t < 0 || t >= p.vocab) ? __builtin_nanf("") : empty ? -__builtin_inff() : (xt - a.m) - ls;
  if (p.lse) { p.lse[2 * row] = empty ? 0.f : a.m; p.lse[2 * row + 1] = empty ? __builtin_inff() : ls; }     // e^(x - m - inf) = 0: no gradient
}
__device__ __forceinline__ void put_top(const LpParams& p, int64_t row, int i, unsigned long long key, const Soft& a) {
  const bool empty = a.m == -__builtin_inff() && a.s == 0.f;
  p.top_logp[row * p.top + i] = empty ? -__builtin_inff() : (key_value(key) - a.m) - logf(a.s);
  p.top_at[row * p.top + i] = key_place(key);
}
template <typename T> __device__ __forceinline__ float token_logit(const LpParams& p, int64_t row) {
  const int64_t t = p.tokens[row];
  return t >= 0 && t < p.vocab ? ldf((const T*)p.x + row * p.ldx + t) : 0.f;
}

// ---- rows that fit a wave's registers ------------------------------------------------------------------------------------
// lane l holds VEC-element accesses l, l + 64, ...
template <typename T, int VEC, int NV>
__global__ __launch_bounds__(256) void lp_wave_kernel(const LpParams p) {
  typedef T vt __attribute__((ext_vector_type(VEC)));
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.ldx;
  float v[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 64 + lane) * VEC;
    if (VEC > 1 && j + VEC <= p.vocab) {
      const vt q = *(const vt*)(x + j);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = (float)q[e];
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = j + e < p.vocab ? ldf(x + j + e) : -__builtin_inff();
    }
  }
  float mx = v[0];
#pragma unroll
  for (int i = 1; i < NV * VEC; ++i) mx = fmaxf(mx, v[i]);
  Soft a = {wave_max64(mx), 0.f, 0.f};
  const float base = safe_max(a.m);
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) soft_add(a, v[i], base);
  a.s = wave_sum64(a.s);
  a.u = wave_sum64(a.u);
  if (lane == 0) finish_row(p, row, a, token_logit<T>(p, row));
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int j = (i * 64 + lane) * VEC + e;
        const unsigned long long key = rank_key(v[i * VEC + e], (unsigned)j);
        if (j < p.vocab && key < last && key > best) best = key;
      }
    last = wave_max_key(best);
    if (lane == 0) put_top(p, row, k, last, a);
  }
}

// ---- a block per row, or per split of a row -----------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void lp_block_kernel(const LpParams p) {
  typedef T vt __attribute__((ext_vector_type(Elt<T>::PIECE)));
  constexpr int VEC = Elt<T>::PIECE;
  __shared__ float sm[4][3], tmax[256];
  __shared__ unsigned long long cand[LP_CAND], best[4], win[LP_MAX_TOP];
  __shared__ int count;
  __shared__ float bound;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x % p.splits);
  const T* x = (const T*)p.x + row * p.ldx;
  const int j0 = split * p.chunk, j1 = j0 + p.chunk < p.vocab ? j0 + p.chunk : p.vocab;
  // head up to the first 16-byte boundary, whole accesses, tail
  int h = (int)(((16 - (uintptr_t)(x + j0) % 16) % 16) / sizeof(T));
  if (h > j1 - j0) h = j1 - j0;
  const int a0 = j0 + h, nvec = (j1 - a0) / VEC, t0 = a0 + nvec * VEC;
  Soft a = {-__builtin_inff(), 0.f, 0.f};
  constexpr int U = 4;
  int i = tid;
  for (; i + (U - 1) * 256 < nvec; i += U * 256) {
    float v[U * VEC];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const vt q = *(const vt*)(x + a0 + (int64_t)(i + k * 256) * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = (float)q[e];
    }
    soft_add_n<U * VEC>(a, v);
  }
  for (; i < nvec; i += 256) {
    float v[VEC];
    const vt q = *(const vt*)(x + a0 + (int64_t)i * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)q[e];
    soft_add_n<VEC>(a, v);
  }
  if (tid < h) { const float v = ldf(x + j0 + tid); soft_add_n<1>(a, &v); }
  if (tid < j1 - t0) { const float v = ldf(x + t0 + tid); soft_add_n<1>(a, &v); }
  const float mine = a.m;
  a = soft_wave(a);
  if (lane == 0) { sm[wave][0] = a.m; sm[wave][1] = a.s; sm[wave][2] = a.u; }
  if (p.top) { tmax[tid] = mine; if (tid == 0) count = 0; }
  __syncthreads();
  {
    Soft q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = Soft{sm[k][0], sm[k][1], sm[k][2]};
    a = soft_join(soft_join(q[0], q[1]), soft_join(q[2], q[3]));
  }
  if (tid == 0) {
    if (p.splits == 1) finish_row(p, row, a, token_logit<T>(p, row));
    else {
      float* o = p.part + (row * p.splits + split) * 4;
      o[0] = a.m; o[1] = a.s; o[2] = a.u;
    }
  }
  if (!p.top) return;
  // The k-th largest of the threads' maxima bounds the k-th largest element from below: k different elements reach it.
  // One wave finds it bit by bit, then everything at or above it is gathered.
  if (wave == 0) {
    unsigned o[4], t = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = (unsigned)(rank_key(tmax[q * 64 + lane], 0) >> 32);
    for (int bit = 31; bit >= 0; --bit) {            // the largest t that at least `top` of the 256 reach
      const unsigned u = t | 1u << bit;
      int n = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) n += __popcll(__ballot(o[q] >= u));
      if (n >= p.top) t = u;
    }
    if (lane == 0) bound = key_value((unsigned long long)t << 32);
  }
  __syncthreads();
  const float low = bound;
  auto gather = [&](float v, unsigned j) {
    if ((v == v ? v : -__builtin_inff()) >= low) {
      const int at = atomicAdd(&count, 1);
      if (at < LP_CAND) cand[at] = rank_key(v, j);
    }
  };
  for (int q = tid; q < nvec; q += 256) {
    const vt w = *(const vt*)(x + a0 + (int64_t)q * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) gather((float)w[e], (unsigned)(a0 + q * VEC + e));
  }
  if (tid < h) gather(ldf(x + j0 + tid), (unsigned)(j0 + tid));
  if (tid < j1 - t0) gather(ldf(x + t0 + tid), (unsigned)(t0 + tid));
  __syncthreads();
  const int n = count;
  if (n >= p.top && n <= LP_CAND) {
    if (wave == 0) best_of(cand, n, p.top, lane, [&](int k, unsigned long long key) { win[k] = key; });
  } else {
    // so many equal values (a constant row), or so few that can be ranked, that the list does not hold the answer: one scan a place
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
      unsigned long long b = 0;
      for (int j = j0 + tid; j < j1; j += 256) {
        const unsigned long long key = rank_key(ldf(x + j), (unsigned)j);
        if (key < last && key > b) b = key;
      }
      b = wave_max_key(b);
      if (lane == 0) best[wave] = b;
      __syncthreads();
      b = best[0];
#pragma unroll
      for (int q = 1; q < 4; ++q) b = best[q] > b ? best[q] : b;
      last = b;
      if (tid == 0) win[k] = last;
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid < p.top) {
    if (p.splits == 1) put_top(p, row, tid, win[tid], a);
    else p.cand[(row * p.splits + split) * p.top + tid] = win[tid];
  }
}

// the splits of one row
#define LP_JOIN 2048
template <typename T> __global__ __launch_bounds__(256) void lp_join_kernel(const LpParams p) {
  __shared__ unsigned long long keys[LP_JOIN];
  const int lane = threadIdx.x & 63, n = p.splits * p.top;
  const int64_t row = blockIdx.x;
  const unsigned long long* c = p.cand + row * n;
  if (n <= LP_JOIN) {
    for (int q = threadIdx.x; q < n; q += 256) keys[q] = c[q];
    __syncthreads();
  }
  if (threadIdx.x >= 64) return;
  Soft a = {-__builtin_inff(), 0.f, 0.f};
  for (int s = lane; s < p.splits; s += 64) {
    const float* o = p.part + (row * p.splits + s) * 4;
    a = soft_join(a, Soft{o[0], o[1], o[2]});
  }
  a = soft_wave(a);
  if (lane == 0) finish_row(p, row, a, token_logit<T>(p, row));
  if (p.top) best_of(n <= LP_JOIN ? keys : c, n, p.top, lane, [&](int k, unsigned long long key) { put_top(p, row, k, key, a); });
}

// ---- backward -----------------------------------------------------------------------------------------------------------
struct LpBwdParams {
  const void* x;
  int64_t ldx;
  const int64_t* tokens;
  int64_t ignore;
  const float *lse, *entropy, *dlogp, *dent;
  void* dx;
  int64_t lddx, rows;
  int vocab, splits, chunk;
};
template <typename T>
__global__ __launch_bounds__(256) void lp_bwd_kernel(const LpBwdParams p, int tpr) {      // tpr: threads of a row (64 or 256)
  constexpr int VEC = Elt<T>::PIECE;
  typedef T vt __attribute__((ext_vector_type(VEC)));
  const int per = 256 / tpr, gl = threadIdx.x % tpr;
  const int64_t unit = blockIdx.x * (int64_t)per + threadIdx.x / tpr;
  const int64_t row = unit / p.splits;
  if (row >= p.rows) return;
  const int split = (int)(unit % p.splits);
  const int j0 = split * p.chunk, j1 = j0 + p.chunk < p.vocab ? j0 + p.chunk : p.vocab;
  const T* x = (const T*)p.x + row * p.ldx;
  T* dx = (T*)p.dx + row * p.lddx;
  const int64_t t = p.tokens[row];
  const bool counts = t != p.ignore && t >= 0 && t < p.vocab;
  const float m = p.lse[2 * row], ls = p.lse[2 * row + 1], h = p.entropy[row];
  const bool empty = ls == __builtin_inff() && m == 0.f;
  const float a = counts && p.dlogp && !empty ? p.dlogp[row] : 0.f, b = p.dent ? p.dent[row] : 0.f;
  auto grad = [&](float v, int j) {
    const float lnp = (v - m) - ls;
    const float e = __expf(lnp);
    const float g = -e * (a + b * (fmaxf(lnp, -200.f) + h));
    return j == (int)t ? g + a : g;
  };
  int hd = (int)(((16 - (uintptr_t)(x + j0) % 16) % 16) / sizeof(T));
  if (hd > j1 - j0) hd = j1 - j0;
  if ((uintptr_t)(dx + j0 + hd) % 16) {              // the two rows are not aligned alike
    for (int j = j0 + gl; j < j1; j += tpr) dx[j] = (T)grad(ldf(x + j), j);
    return;
  }
  const int a0 = j0 + hd, nvec = (j1 - a0) / VEC, t0 = a0 + nvec * VEC;
  for (int i = gl; i < nvec; i += tpr) {
    const vt q = *(const vt*)(x + a0 + (int64_t)i * VEC);
    vt o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)grad((float)q[e], a0 + i * VEC + e);
    *(vt*)(dx + a0 + (int64_t)i * VEC) = o;
  }
  if (gl < hd) dx[j0 + gl] = (T)grad(ldf(x + j0 + gl), j0 + gl);
  if (gl < j1 - t0) dx[t0 + gl] = (T)grad(ldf(x + t0 + gl), t0 + gl);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// A row is split when the rows alone are too few to fill the chip; a split keeps at least 2048 elements, so that joining
// stays small beside reading.
static void lp_split(int64_t rows, int vocab, int* splits, int* chunk) {
  int64_t s = vg_ceil_div(512, rows);
  const int64_t most = vg_ceil_div(vocab, 2048);
  if (s > most) s = most;
  if (s < 1) s = 1;
  *chunk = (int)(vg_ceil_div(vg_ceil_div(vocab, s), 8) * 8);
  *splits = (int)vg_ceil_div(vocab, *chunk);
}
static int lp_check(const char* what, int64_t rows, int vocab, int64_t ldx, int top, int dtype) {
  VG_REQUIRE(dtype == VG_F32 || dtype == VG_BF16, "%s: dtype %d", what, dtype);
  VG_REQUIRE(rows >= 0 && rows < (1LL << 31) && vocab >= 1 && vocab <= (1 << 30) && ldx >= vocab, "%s: %ld rows of %d logits, stride %ld",
             what, (long)rows, vocab, (long)ldx);
  VG_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, "%s: %d alternatives of %d (at most %d)", what, top, vocab, LP_MAX_TOP);
  return VG_OK;
}
static bool lp_regs(int vocab) { return vocab <= 64 * 32; }      // a row in the registers of a wave

extern "C" size_t vg_token_logprobs_ws_bytes(int64_t rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0 || lp_regs(vocab)) return 0;
  int s, c;
  lp_split(rows, vocab, &s, &c);
  return s == 1 ? 0 : (size_t)rows * s * (4 * sizeof(float) + (size_t)top * 8);
}

template <typename T> static void lp_launch(const LpParams& p, hipStream_t st) {
  if (lp_regs(p.vocab)) {
    constexpr int V = Elt<T>::PIECE;
    const dim3 grid((unsigned)vg_ceil_div(p.rows, 4));
    const bool vec = (uintptr_t)p.x % 16 == 0 && (p.ldx * sizeof(T)) % 16 == 0;
#define LP_CASE(VEC, NV) \
  if (p.vocab <= 64 * VEC * NV) { hipLaunchKernelGGL((lp_wave_kernel<T, VEC, NV>), grid, dim3(256), 0, st, p); return; }
    if (vec) {
      if constexpr (V == 4) { LP_CASE(4, 1) LP_CASE(4, 2) LP_CASE(4, 4) LP_CASE(4, 8) }
      else { LP_CASE(8, 1) LP_CASE(8, 2) LP_CASE(8, 4) }
    } else { LP_CASE(1, 4) LP_CASE(1, 8) LP_CASE(1, 16) LP_CASE(1, 32) }
#undef LP_CASE
    return;
  }
  hipLaunchKernelGGL(lp_block_kernel<T>, dim3((unsigned)(p.rows * p.splits)), dim3(256), 0, st, p);
  if (p.splits > 1) hipLaunchKernelGGL(lp_join_kernel<T>, dim3((unsigned)p.rows), dim3(256), 0, st, p);
}

extern "C" int vg_token_logprobs_fwd(const void* logits, int64_t ldx, const int64_t* tokens, int64_t ignore, int64_t rows, int vocab,
                                     int top, float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_at, void* ws,
                                     int dtype, void* stream) {
  if (int rc = lp_check("token_logprobs_fwd", rows, vocab, ldx, top, dtype)) return rc;
  if (rows == 0) return VG_OK;
  VG_REQUIRE(logits && tokens && logp && entropy && (!top || (top_logp && top_at)), "token_logprobs_fwd: null pointer");
  VG_REQUIRE(ws || vg_token_logprobs_ws_bytes(rows, vocab, top) == 0, "token_logprobs_fwd: needs a workspace");
  LpParams p = {logits, ldx, tokens, ignore, rows, vocab, top, 1, 0, logp, entropy, lse, top_logp, top_at, nullptr, nullptr};
  lp_split(rows, vocab, &p.splits, &p.chunk);
  p.cand = (unsigned long long*)ws;                  // 8-byte values first
  p.part = (float*)((char*)ws + (size_t)rows * p.splits * top * 8);
  if (dtype == VG_BF16) lp_launch<bf16_t>(p, (hipStream_t)stream);
  else lp_launch<float>(p, (hipStream_t)stream);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

extern "C" int vg_token_logprobs_bwd(const void* logits, int64_t ldx, const int64_t* tokens, int64_t ignore, const float* lse,
                                     const float* entropy, const float* dlogp, const float* dent, void* dx, int64_t lddx, int64_t rows,
                                     int vocab, int dtype, void* stream) {
  if (int rc = lp_check("token_logprobs_bwd", rows, vocab, ldx, 0, dtype)) return rc;
  if (rows == 0) return VG_OK;
  VG_REQUIRE(logits && tokens && lse && entropy && dx && lddx >= vocab, "token_logprobs_bwd: null pointer or a short row stride");
  LpBwdParams p = {logits, ldx, tokens, ignore, lse, entropy, dlogp, dent, dx, lddx, rows, vocab, 1, 0};
  // a wave per row while the row is short; otherwise blocks, each with at most 32 KB of a row
  const int tpr = vocab <= 4096 ? 64 : 256;
  p.chunk = tpr == 64 ? (int)(vg_ceil_div(vocab, 8) * 8) : (1 << 14);
  p.splits = (int)vg_ceil_div(vocab, p.chunk);
  const int64_t units = rows * p.splits;
  const int64_t blocks = vg_ceil_div(units, 256 / tpr);
  VG_REQUIRE(blocks < (1LL << 31), "token_logprobs_bwd: %ld rows of %d logits are too many for one launch", (long)rows, vocab);
  if (dtype == VG_BF16) hipLaunchKernelGGL(lp_bwd_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p, tpr);
  else hipLaunchKernelGGL(lp_bwd_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p, tpr);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

// Log probabilities of given tokens under rows of logits, with the entropy and the best alternatives, and their gradient.
//   m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m):  logp = (x_t - m) - ln s,  H = ln s - u / s
//   dx_j = dlogp ([j = t] - p_j) - dH p_j (ln p_j + H),  p_j = e^(x_j - lse)
// Bound by memory: the forward reads the logits once, keeping (m, s, u) as running values that are rescaled when a larger
// maximum arrives; the backward reads them once more and writes the gradient (16384 x 8192 bf16, one after the other: 52 and
// 83 us, 805 MB at 6.0 TB/s, a part of the logits from the last-level cache).  Sums are f32; exponents are of x - m <= 0.
// Masked logits (-inf) have p = 0, so by the formula no gradient, except a masked token in a row that allows others: logp -inf,
// and dlogp at its place.  A row of nothing but -inf has no distribution: logp -inf, H 0, gradient 0.  A
// NaN or +inf in a row makes its logp, H and gradient NaN.  tokens[r] == ignore: logp 0 and no gradient through logp; any
// other token outside [0, vocab) gives logp NaN and no gradient through logp (it is never used as an index).
#include "common.h"
#include "rows.h"

#define LP_MAX_TOP 32
#define LP_CAND 512        // candidates a block (a wave: a quarter) can hold for the selection of the best

template <typename T> __device__ __forceinline__ float ldf(const T* p) { return (float)*p; }

// A set of logits: m (its maximum), s = sum 2^d and u = sum 2^d d with d = x log2 e - c, c = m log2 e as rounded to f32: one
// fused multiply-add and one exponential an element.  The rounding of c is the same in every d, so it cancels in d - log2 s; it
// grows with |m|, and 2^(it) has to fit the sums: from |m| = LP_FAR (2^20: 2^-4 there) up, d = (x - m) log2 e, whose rounding is
// that of the distance alone.  Masked elements have d = -inf: clamped where it multiplies, since 0 * -inf is NaN (2^-290 is 0 in f32).
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f
#define LP_FAR 0x1p20f
#define LP_WIDE 2e38f      // x log2 e stays in range below it
struct Soft { float m, s, u; };
__device__ __forceinline__ float soft_base(float m) { return m == -__builtin_inff() ? 0.f : m; }
__device__ __forceinline__ float soft_d(float x, float base) {
  return fabsf(base) < LP_FAR ? fmaf(x, LP_LOG2E, -(base * LP_LOG2E)) : (x - base) * LP_LOG2E;
}
// base log2 e - c, exactly: what every d about this base holds beside (x - base) log2 e
__device__ __forceinline__ float soft_residual(float base) { return fabsf(base) < LP_FAR ? fmaf(base, LP_LOG2E, -(base * LP_LOG2E)) : 0.f; }
// the same set about a larger maximum; the residual of the old base leaves its sums and that of the new one enters, or a set
// that is joined from sets about near and far maxima would not be one sum
__device__ __forceinline__ Soft soft_about(const Soft& a, float m) {
  const float b = soft_base(m);
  const float d = fmaxf((a.m - b) * LP_LOG2E + (soft_residual(b) - soft_residual(a.m)), -290.f), e = __builtin_amdgcn_exp2f(d);
  return Soft{m, a.s * e, e * (a.u + d * a.s)};
}
// (m, s, u) of two disjoint sets
__device__ __forceinline__ Soft soft_join(const Soft& a, const Soft& b) {
  const float m = fmaxf(a.m, b.m);
  const Soft p = soft_about(a, m), q = soft_about(b, m);
  return Soft{m, p.s + q.s, p.u + q.u};
}
template <int N> __device__ __forceinline__ void soft_add(Soft& a, const float* x) {
  const float base = soft_base(a.m);
  const bool near = fabsf(base) < LP_FAR;
  const float c = near ? base * LP_LOG2E : 0.f;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = x[i];
  if (!near) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] -= base;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = fmaf(y[i], LP_LOG2E, -c), e = __builtin_amdgcn_exp2f(d);
    a.s += e;
    a.u += e * fmaxf(d, -290.f);
  }
}
template <int N> __device__ __forceinline__ void soft_add_n(Soft& a, const float* x) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  if (m > a.m) a = soft_about(a, m);
  soft_add<N>(a, x);
}
__device__ __forceinline__ Soft soft_wave(const Soft& a) {
  const Soft b = soft_about(a, wave_max64(a.m));
  return Soft{b.m, wave_sum64(b.s), wave_sum64(b.u)};
}
__device__ __forceinline__ bool soft_empty(const Soft& a) { return a.m == -__builtin_inff() && a.s == 0.f; }

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
  const unsigned hi = wave_umax64((unsigned)(k >> 32));       // the best value, then the best place among those that have it
  const unsigned lo = wave_umax64((unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
  return ((unsigned long long)hi << 32) | lo;
}

// the `top` largest of n different keys (0: none), to put(k, key), by one wave
template <typename F> __device__ __forceinline__ void best_of(const unsigned long long* keys, int n, int top, int lane, F put) {
  if (n <= 64) {                                     // each lane counts the keys above its own
    const unsigned long long mine = lane < n ? keys[lane] : 0;
    int above = 0;
    for (int q = 0; q < n; ++q) {
      const unsigned long long o = (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(mine >> 32), q) << 32 |
                                   (unsigned)__builtin_amdgcn_readlane((int)mine, q);
      above += o > mine;
    }
    if (mine && above < top) put(above, mine);
    return;
  }
  constexpr int R = 8;                               // the first 512 in registers
  unsigned long long mine[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mine[r] = r * 64 + lane < n ? keys[r * 64 + lane] : 0;
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long b = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (mine[r] < last && mine[r] > b) b = mine[r];
    for (int q = R * 64 + lane; q < n; q += 64)
      if (keys[q] < last && keys[q] > b) b = keys[q];
    last = wave_max_key(b);
    if (lane == 0 && last) put(k, last);
    if (!last) break;
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

// ln p of a logit: (d - log2 s) ln 2, with d as it was summed.  About a far maximum, and of a logit that is far down, d can
// overflow where ln p does not: x - m - ln s (s about a far maximum has no residual; beside |x| >= LP_WIDE one does not count)
__device__ __forceinline__ float soft_lnp(float x, const Soft& a) {
  const float l2 = log2f(a.s);
  return fabsf(a.m) < LP_FAR && fabsf(x) < LP_WIDE ? (soft_d(x, a.m) - l2) * LP_LN2 : (x - a.m) - l2 * LP_LN2;
}
__device__ __forceinline__ void finish_row(const LpParams& p, int64_t row, const Soft& a, float xt) {
  const bool empty = soft_empty(a);
  const float l2 = log2f(a.s);
  const int64_t t = p.tokens[row];
  p.entropy[row] = empty ? 0.f : (l2 - a.u / a.s) * LP_LN2;
  p.logp[row] = t == p.ignore ? 0.f : (t < 0 || t >= p.vocab) ? __builtin_nanf("") : empty ? -__builtin_inff() : soft_lnp(xt, a);
  if (p.lse) { p.lse[2 * row] = empty ? 0.f : a.m; p.lse[2 * row + 1] = empty ? __builtin_inff() : l2; }     // 2^(d - inf) = 0: no gradient
}
__device__ __forceinline__ void put_top(const LpParams& p, int64_t row, int i, unsigned long long key, const Soft& a) {
  p.top_logp[row * p.top + i] = soft_empty(a) ? -__builtin_inff() : soft_lnp(key_value(key), a);
  p.top_at[row * p.top + i] = key_place(key);
}
template <typename T> __device__ __forceinline__ float token_logit(const LpParams& p, int64_t row) {
  const int64_t t = p.tokens[row];
  return t >= 0 && t < p.vocab ? ldf((const T*)p.x + row * p.ldx + t) : 0.f;
}

// ---- rows that fit a wave's registers ------------------------------------------------------------------------------------
// lane l holds 16-byte accesses l, l + 64, ..., aligned to an element only (the machine's global memory instructions take that)
// GL lanes share a row (short rows: several to a wave; 65536 x 128 bf16: 18 us with a wave each, 7 with 16 lanes)
template <int GL, typename V, typename F> __device__ __forceinline__ V group_fold(V v, F f) {
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) v = f(v, (V)__shfl_xor(v, o, 64));
  return v;
}
template <int GL> __device__ __forceinline__ float group_max(float v) {
  if constexpr (GL == 64) return wave_max64(v);
  else return group_fold<GL>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int GL> __device__ __forceinline__ float group_sum(float v) {
  if constexpr (GL == 64) return wave_sum64(v);
  else return group_fold<GL>(v, [](float a, float b) { return a + b; });
}
template <int GL> __device__ __forceinline__ unsigned long long group_max_key(unsigned long long k) {
  if constexpr (GL == 64) return wave_max_key(k);
  else {
    auto larger = [](unsigned a, unsigned b) { return a > b ? a : b; };
    const unsigned hi = group_fold<GL>((unsigned)(k >> 32), larger);
    return ((unsigned long long)hi << 32) | group_fold<GL>((unsigned)(k >> 32) == hi ? (unsigned)k : 0u, larger);
  }
}
template <typename T, int GL, int NV>
__global__ __launch_bounds__(256) void lp_wave_kernel(const LpParams p) {
  constexpr int VEC = Elt<T>::PIECE;
  typedef T vt __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  const int lane = threadIdx.x % GL;
  const int64_t row = blockIdx.x * (int64_t)(256 / GL) + threadIdx.x / GL;
  if (row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.ldx;
  float v[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * GL + lane) * VEC;
    if (j + VEC <= p.vocab) {
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
  Soft a = {group_max<GL>(mx), 0.f, 0.f};
  soft_add<NV * VEC>(a, v);
  a.s = group_sum<GL>(a.s);
  a.u = group_sum<GL>(a.u);
  if (lane == 0) finish_row(p, row, a, token_logit<T>(p, row));
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int j = (i * GL + lane) * VEC + e;
        const unsigned long long key = rank_key(v[i * VEC + e], (unsigned)j);
        if (j < p.vocab && key < last && key > best) best = key;
      }
    last = group_max_key<GL>(best);
    if (lane == 0) put_top(p, row, k, last, a);
  }
}

// ---- a block per row, or per split of a row -----------------------------------------------------------------------------
// A unit (a row, or a split of one) belongs to a team: a wave, or the four waves of a block.
template <int TEAM> __device__ __forceinline__ void team_sync() {
  if constexpr (TEAM > 64) __syncthreads();
  else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}
template <int TEAM> struct LpLists {                 // of one team, in LDS
  static constexpr int CAND = LP_CAND * TEAM / 256;
  unsigned long long cand[CAND], best[4], win[LP_MAX_TOP];
  float tmax[TEAM];
  unsigned char who[TEAM];           // threads whose elements are looked through once more
  int count, whos;
  float bound;
};
template <typename T> struct LpUnit { const T* x; int64_t row; int split, j0, j1, a0, nvec; };

// the best of one unit; mine: the maximum of this thread's elements, a: the unit's sums (its row's, where it is one)
template <typename T, int TEAM>
__device__ void lp_best(const LpParams& p, const LpUnit<T>& u, LpLists<TEAM>& l, float mine, const Soft& a) {
  constexpr int VEC = Elt<T>::PIECE;
  typedef T vt __attribute__((ext_vector_type(VEC)));
  const int tid = threadIdx.x % TEAM, lane = tid & 63, wave = tid >> 6, h = u.a0 - u.j0, t0 = u.a0 + u.nvec * VEC;
  l.tmax[tid] = mine;
  if (tid == 0) l.count = l.whos = 0;
  if (tid < LP_MAX_TOP) l.win[tid] = 0;
  team_sync<TEAM>();
  // The k-th largest of the threads' maxima bounds the k-th largest element from below: k different elements reach it.
  // One wave finds it bit by bit, then everything at or above it is gathered: out of the elements of those threads alone whose
  // maximum reaches it, dealt to the whole team, so that the second look costs one access a thread and not one more pass
  // (560 x 51415 f32, top 8: 47 -> 26 us).
  if (wave == 0) {
    unsigned o[TEAM / 64], t = 0;
#pragma unroll
    for (int q = 0; q < TEAM / 64; ++q) o[q] = (unsigned)(rank_key(l.tmax[q * 64 + lane], 0) >> 32);
    for (int bit = 31; bit >= 0; --bit) {            // the largest t that at least `top` of the maxima reach
      const unsigned v = t | 1u << bit;
      int n = 0;
#pragma unroll
      for (int q = 0; q < TEAM / 64; ++q) n += __popcll(__ballot(o[q] >= v));
      if (n >= p.top) t = v;
    }
    if (lane == 0) l.bound = key_value((unsigned long long)t << 32);
  }
  team_sync<TEAM>();
  const float low = l.bound;
  bool above = low == -__builtin_inff();             // only what is larger than the bound: its equals may be too many to list
  int n;
  for (;;) {
    auto gather = [&](float v, unsigned j) {
      if (above ? v > low : v >= low) {
        const int at = atomicAdd(&l.count, 1);
        if (at < l.CAND) l.cand[at] = rank_key(v, j);
      }
    };
    auto look = [&](int q) {
      const vt v = *(const vt*)(u.x + u.a0 + (int64_t)q * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) gather((float)v[e], (unsigned)(u.a0 + q * VEC + e));
    };
    const bool holds = above ? mine > low : mine >= low;
    const int each = (u.nvec + TEAM - 1) / TEAM;     // accesses of a thread
    if (each <= 2) {                                 // nothing to deal
      for (int q = holds ? tid : u.nvec; q < u.nvec; q += TEAM) look(q);
    } else {
      if (holds) l.who[atomicAdd(&l.whos, 1)] = (unsigned char)tid;
      team_sync<TEAM>();
      for (int it = tid, items = l.whos * each; it < items; it += TEAM) {
        const int w = it / each, q = (it - w * each) * TEAM + l.who[w];
        if (q < u.nvec) look(q);
      }
    }
    if (tid < h) gather(ldf(u.x + u.j0 + tid), (unsigned)(u.j0 + tid));
    if (tid < u.j1 - t0) gather(ldf(u.x + t0 + tid), (unsigned)(t0 + tid));
    team_sync<TEAM>();
    n = l.count;
    if (above || n <= l.CAND) break;
    above = true;                                    // a row of many equal values
    team_sync<TEAM>();
    if (tid == 0) l.count = l.whos = 0;
    team_sync<TEAM>();
  }
  if (n <= l.CAND) {
    if (wave == 0) {
      // of the bound's equals (of -inf: all that is masked), the first ones fill the places that are left
      constexpr int AHEAD = 8;                       // loads in flight: the first equal may be far
      for (int base = u.j0; n < p.top && base < u.j1; base += 64 * AHEAD) {
        float v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = base + k * 64 + lane < u.j1 ? ldf(u.x + base + k * 64 + lane) : 0.f;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int j = base + k * 64 + lane;
          const bool equal = j < u.j1 && (v[k] == v[k] ? v[k] : -__builtin_inff()) == low;
          const unsigned long long which = __ballot(equal);
          const int at = n + __popcll(which & ((1ull << lane) - 1));
          if (equal && at < p.top) l.cand[at] = rank_key(v[k], (unsigned)j);
          n = min(n + __popcll(which), p.top);
        }
      }
      team_sync<64>();
      best_of(l.cand, n, p.top, lane, [&](int k, unsigned long long key) { l.win[k] = key; });
    }
  } else {
    // a few threads hold more above the bound than the list does (values that repeat with the threads' stride): one scan a place
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
      unsigned long long b = 0;
      for (int j = u.j0 + tid; j < u.j1; j += TEAM) {
        const unsigned long long key = rank_key(ldf(u.x + j), (unsigned)j);
        if (key < last && key > b) b = key;
      }
      b = wave_max_key(b);
      if constexpr (TEAM > 64) {
        if (lane == 0) l.best[wave] = b;
        __syncthreads();
        b = l.best[0];
#pragma unroll
        for (int q = 1; q < 4; ++q) b = l.best[q] > b ? l.best[q] : b;
        __syncthreads();
      }
      last = b;
      if (tid == 0) l.win[k] = last;
    }
  }
  team_sync<TEAM>();
  if (tid < p.top) {
    if (p.splits == 1) put_top(p, u.row, tid, l.win[tid], a);
    else p.cand[(u.row * p.splits + u.split) * p.top + tid] = l.win[tid];
  }
}

// The logits of a thread come in batches of U 16-byte accesses; the next batch is on its way while one is summed.
template <typename T, int U, int TEAM>
__global__ __launch_bounds__(256) void lp_row_kernel(const LpParams p) {
  constexpr int VEC = Elt<T>::PIECE;
  typedef T vt __attribute__((ext_vector_type(VEC)));
  __shared__ float sm[4][3];
  __shared__ LpLists<TEAM> lists[256 / TEAM];
  const int tid = threadIdx.x % TEAM, lane = tid & 63, wave = tid >> 6;
  const int64_t id = blockIdx.x * (int64_t)(256 / TEAM) + threadIdx.x / TEAM;
  if (id >= p.rows * p.splits) return;               // a whole team: a block has one team or no barriers
  LpUnit<T> u;
  u.row = id / p.splits;
  u.split = (int)(id % p.splits);
  u.x = (const T*)p.x + u.row * p.ldx;
  u.j0 = u.split * p.chunk;
  u.j1 = u.j0 + p.chunk < p.vocab ? u.j0 + p.chunk : p.vocab;
  const int h = (int)(((16 - (uintptr_t)(u.x + u.j0) % 16) % 16) / sizeof(T));      // elements before the first 16-byte boundary
  u.a0 = u.j0 + (h < u.j1 - u.j0 ? h : u.j1 - u.j0);
  u.nvec = (u.j1 - u.a0) / VEC;
  vt next[U];
  auto fetch = [&](int at) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = at + k * TEAM + tid;
      if (i < u.nvec) next[k] = *(const vt*)(u.x + u.a0 + (int64_t)i * VEC);
      else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) next[k][e] = (T)(-__builtin_inff());
      }
    }
  };
  Soft a = {-__builtin_inff(), 0.f, 0.f};
  fetch(0);
  for (int at = U * TEAM;; at += U * TEAM) {
    float v[U * VEC];
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = (float)next[k][e];
    if (at < u.nvec) fetch(at);
    soft_add_n<U * VEC>(a, v);
    if (at >= u.nvec) break;
  }
  const int t0 = u.a0 + u.nvec * VEC;
  if (tid < u.a0 - u.j0) { const float v = ldf(u.x + u.j0 + tid); soft_add_n<1>(a, &v); }
  if (tid < u.j1 - t0) { const float v = ldf(u.x + t0 + tid); soft_add_n<1>(a, &v); }
  const float mine = a.m;
  a = soft_wave(a);
  if constexpr (TEAM > 64) {
    if (lane == 0) { sm[wave][0] = a.m; sm[wave][1] = a.s; sm[wave][2] = a.u; }
    __syncthreads();
    Soft q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = Soft{sm[k][0], sm[k][1], sm[k][2]};
    a = soft_join(soft_join(q[0], q[1]), soft_join(q[2], q[3]));
  }
  if (tid == 0) {
    if (p.splits == 1) finish_row(p, u.row, a, token_logit<T>(p, u.row));
    else {
      float* o = p.part + (u.row * p.splits + u.split) * 4;
      o[0] = a.m; o[1] = a.s; o[2] = a.u;
    }
  }
  if (p.top) lp_best<T, TEAM>(p, u, lists[threadIdx.x / TEAM], mine, a);
}

// The splits of one row.  Its parts (memory, selection, sums) run side by side on the block's waves: each wave takes a quarter
// of the splits' best, the last wave fetches the token's logit meanwhile.
template <typename T> __global__ __launch_bounds__(256) void lp_join_kernel(const LpParams p) {
  __shared__ unsigned long long some[4 * LP_MAX_TOP], win[LP_MAX_TOP];
  __shared__ float sums[3], xt;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = p.splits * p.top;
  const int64_t row = blockIdx.x;
  if (threadIdx.x == 255) xt = token_logit<T>(p, row);
  if (p.top) {
    const int per = (n + 3) / 4, lo = wave * per < n ? wave * per : n, hi = lo + per < n ? lo + per : n;
    if (lane < p.top) some[wave * p.top + lane] = 0;          // a quarter may hold fewer
    __builtin_amdgcn_wave_barrier();
    best_of(p.cand + row * n + lo, hi - lo, p.top, lane, [&](int k, unsigned long long key) { some[wave * p.top + k] = key; });
  }
  if (wave == 0) {
    Soft a = {-__builtin_inff(), 0.f, 0.f};
    for (int s = lane; s < p.splits; s += 64) {
      const f32x4 o = *(const f32x4*)(p.part + (row * p.splits + s) * 4);
      a = soft_join(a, Soft{o[0], o[1], o[2]});
    }
    a = soft_wave(a);
    if (lane == 0) { sums[0] = a.m; sums[1] = a.s; sums[2] = a.u; }
  }
  __syncthreads();
  const Soft a = {sums[0], sums[1], sums[2]};
  if (threadIdx.x == 64) finish_row(p, row, a, xt);
  if (!p.top) return;
  if (wave == 0) {
    best_of(some, 4 * p.top, p.top, lane, [&](int k, unsigned long long key) { win[k] = key; });
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (lane < p.top) put_top(p, row, lane, win[lane], a);
  }
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
// STREAM (logits and gradient take more than LP_STREAM bytes, most of the last-level cache): stores that do not allocate there
// leave it to the logits, and the copy of the gradient that follows does not wait for their eviction.  Forward, backward and a
// read of the gradient, 16384 x 8192 bf16: 251 us so, 262 otherwise; 6000 x 8192: 94 and 100; 4096 x 8192, which fits: 70 and 66.
#define LP_STREAM (160ll << 20)
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void lp_bwd_kernel(const LpBwdParams p, int tpr) {      // tpr: threads of a row (8 .. 64 or 256)
  constexpr int VEC = Elt<T>::PIECE;
  typedef T vt __attribute__((ext_vector_type(VEC)));
  typedef T ut __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));      // the gradient's rows may be aligned otherwise
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
  const float m = p.lse[2 * row], l2 = p.lse[2 * row + 1], h = p.entropy[row];
  const bool empty = l2 == __builtin_inff() && m == 0.f;
  const float a = counts && p.dlogp && !empty ? p.dlogp[row] : 0.f, b = p.dent ? p.dent[row] : 0.f;
  auto grad = [&](float v, int j) {
    const float d = soft_d(v, m) - l2, e = __builtin_amdgcn_exp2f(d);
    const float g = -e * (a + b * (fmaxf(d, -290.f) * LP_LN2 + h));
    return j == (int)t ? g + a : g;
  };
  int hd = (int)(((16 - (uintptr_t)(x + j0) % 16) % 16) / sizeof(T));
  if (hd > j1 - j0) hd = j1 - j0;
  const int a0 = j0 + hd, nvec = (j1 - a0) / VEC, t0 = a0 + nvec * VEC;
  for (int i = gl; i < nvec; i += tpr) {
    const vt q = *(const vt*)(x + a0 + (int64_t)i * VEC);
    ut o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)grad((float)q[e], a0 + i * VEC + e);
    if (STREAM) __builtin_nontemporal_store(o, (ut*)(dx + a0 + (int64_t)i * VEC));
    else *(ut*)(dx + a0 + (int64_t)i * VEC) = o;
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

static size_t lp_keys_bytes(int64_t rows, int splits, int top) { return ((size_t)rows * splits * top * 8 + 15) / 16 * 16; }
extern "C" size_t vg_token_logprobs_ws_bytes(int64_t rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0 || lp_regs(vocab)) return 0;
  int s, c;
  lp_split(rows, vocab, &s, &c);
  return s == 1 ? 0 : (size_t)rows * s * 4 * sizeof(float) + lp_keys_bytes(rows, s, top);
}

static const int64_t LP_WAVE_UNITS = 2048;          // two waves a SIMD
template <typename T> static int lp_launch(const LpParams& p, hipStream_t st) {
  if (lp_regs(p.vocab)) {
#define LP_CASE(GL, NV)                                                                              \
  if (p.vocab <= GL * Elt<T>::PIECE * NV) {                                                          \
    const int64_t blocks = vg_ceil_div(p.rows, 256 / GL);                                            \
    VG_GRID_CHECK("token_logprobs_fwd", blocks, 256);                                                \
    hipLaunchKernelGGL((lp_wave_kernel<T, GL, NV>), dim3((unsigned)blocks), dim3(256), 0, st, p);    \
    VG_LAUNCH_CHECK();                                                                               \
    return VG_OK;                                                                                    \
  }
    LP_CASE(8, 1) LP_CASE(16, 1) LP_CASE(32, 1) LP_CASE(64, 1) LP_CASE(64, 2) LP_CASE(64, 4)
    if constexpr (sizeof(T) == 4) { LP_CASE(64, 8) }
#undef LP_CASE
  }
  // Many rows: a wave each, which leaves no barrier between loads and sums, two accesses a batch (16384 x 8192 bf16: 51 us,
  // 5.2 TB/s; a batch of four 72, since its registers halve the waves).  Few: a block each, with as many accesses in a batch
  // as a unit has for each thread.
  const int64_t units = p.rows * p.splits, per = vg_ceil_div(p.chunk < p.vocab ? p.chunk : p.vocab, 256 * Elt<T>::PIECE);
  VG_GRID_CHECK("token_logprobs_fwd", units >= LP_WAVE_UNITS ? vg_ceil_div(units, 4) : units, 256);
  if (units >= LP_WAVE_UNITS) hipLaunchKernelGGL((lp_row_kernel<T, 2, 64>), dim3((unsigned)vg_ceil_div(units, 4)), dim3(256), 0, st, p);
  else if (per == 1) hipLaunchKernelGGL((lp_row_kernel<T, 1, 256>), dim3((unsigned)units), dim3(256), 0, st, p);
  else if (per == 2) hipLaunchKernelGGL((lp_row_kernel<T, 2, 256>), dim3((unsigned)units), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((lp_row_kernel<T, 4, 256>), dim3((unsigned)units), dim3(256), 0, st, p);
  if (p.splits > 1) hipLaunchKernelGGL(lp_join_kernel<T>, dim3((unsigned)p.rows), dim3(256), 0, st, p);
  VG_LAUNCH_CHECK();
  return VG_OK;
}

extern "C" int vg_token_logprobs_fwd(const void* logits, int64_t ldx, const int64_t* tokens, int64_t ignore, int64_t rows, int vocab,
                                     int top, float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_at, void* ws,
                                     int dtype, void* stream) {
  if (int rc = lp_check("token_logprobs_fwd", rows, vocab, ldx, top, dtype)) return rc;
  if (rows == 0) return VG_OK;
  VG_REQUIRE(logits && tokens && logp && entropy && (!top || (top_logp && top_at)), "token_logprobs_fwd: null pointer");
  VG_REQUIRE((uintptr_t)ws % 16 == 0 && (ws || vg_token_logprobs_ws_bytes(rows, vocab, top) == 0),
             "token_logprobs_fwd: needs a workspace, aligned to 16 bytes");
  LpParams p = {logits, ldx, tokens, ignore, rows, vocab, top, 1, 0, logp, entropy, lse, top_logp, top_at, nullptr, nullptr};
  lp_split(rows, vocab, &p.splits, &p.chunk);
  p.cand = (unsigned long long*)ws;                  // 8-byte values first
  p.part = (float*)((char*)ws + lp_keys_bytes(rows, p.splits, top));
  return dtype == VG_BF16 ? lp_launch<bf16_t>(p, (hipStream_t)stream) : lp_launch<float>(p, (hipStream_t)stream);
}

extern "C" int vg_token_logprobs_bwd(const void* logits, int64_t ldx, const int64_t* tokens, int64_t ignore, const float* lse,
                                     const float* entropy, const float* dlogp, const float* dent, void* dx, int64_t lddx, int64_t rows,
                                     int vocab, int dtype, void* stream) {
  if (int rc = lp_check("token_logprobs_bwd", rows, vocab, ldx, 0, dtype)) return rc;
  if (rows == 0) return VG_OK;
  VG_REQUIRE(logits && tokens && lse && entropy && dx && lddx >= vocab, "token_logprobs_bwd: null pointer or a short row stride");
  LpBwdParams p = {logits, ldx, tokens, ignore, lse, entropy, dlogp, dent, dx, lddx, rows, vocab, 1, 0};
  // up to a wave per row while the row is short (65536 x 128 bf16: 24 us with a wave, 10 with 16 lanes); otherwise blocks,
  // each with at most 16384 elements of a row
  int tpr = vocab <= 4096 ? 64 : 256;
  while (tpr > 8 && vocab <= tpr / 2 * (16 / vg_elt_size(dtype))) tpr /= 2;
  p.chunk = tpr <= 64 ? (int)(vg_ceil_div(vocab, 8) * 8) : (1 << 14);
  p.splits = (int)vg_ceil_div(vocab, p.chunk);
  const int64_t units = rows * p.splits;
  const int64_t blocks = vg_ceil_div(units, 256 / tpr);
  VG_GRID_CHECK("token_logprobs_bwd", blocks, 256);
  const bool stream_out = rows * (int64_t)vocab * 2 * vg_elt_size(dtype) > LP_STREAM;
#define LP_BWD(T, S) hipLaunchKernelGGL((lp_bwd_kernel<T, S>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p, tpr)
  if (dtype == VG_BF16) { if (stream_out) LP_BWD(bf16_t, true); else LP_BWD(bf16_t, false); }
  else { if (stream_out) LP_BWD(float, true); else LP_BWD(float, false); }
#undef LP_BWD
  VG_LAUNCH_CHECK();
  return VG_OK;
}

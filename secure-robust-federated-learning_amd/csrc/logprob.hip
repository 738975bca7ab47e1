// k14 — log probabilities of given tokens, with the entropy and the top
// alternatives of every row, and the logits' gradient.
//
// One pass over a row keeps, per thread, the running maximum m and
//   s = sum e^{x - m},   u = sum e^{x - m} (x - m),
// joined over threads and waves by
//   (m, s, u) + (m', s', u'):  with M = max(m, m'), d = m - M, f = e^d:
//   s f + ...,  (u + s d) f + ...
// so that  lse = m + log s,  logp = (x_target - m) - log s,  entropy = log s - u / s
// without a difference of large numbers.  lse is held as two floats, the rounded
// sum and what its rounding left, so that x - lse keeps the digits of log s however
// large the logits are (rows of float32's lowest value: log s next to 3.4e38).
#include <type_traits>

#include "lm_common.hpp"

namespace sra {

unsigned int logprob_row_faults(bool reset) { return tu_row_faults(reset); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
// differences from the maximum below this have e^d = 0; clamping them keeps
// 0 * d from becoming NaN for -inf logits
constexpr float kFarBelow = -1.0e4f;

__device__ __forceinline__ float fast_exp(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

struct Stats {
  float m, s, u;
};

__device__ __forceinline__ void rescale(Stats& a, float M) {
  const float d = a.m - M;
  const float f = fast_exp(d);
  a.u = (a.u + a.s * fmaxf(d, kFarBelow)) * f;
  a.s *= f;
  a.m = M;
}

__device__ __forceinline__ void join(Stats& a, Stats b) {
  const float M = __builtin_elementwise_maximum(a.m, b.m);   // keeps a NaN
  rescale(a, M);
  rescale(b, M);
  a.s += b.s;
  a.u += b.u;
}

// m + log s in two floats, exactly: the larger addend comes back from the sum
// without an error, and the other less that is what the rounding left.
struct Lse {
  float hi, lo;
  __device__ __forceinline__ float below(float x) const { return (x - hi) - lo; }
};

__device__ __forceinline__ Lse lse_of(float m, float ls) {
  const float hi = m + ls;
  return {hi, fabsf(m) >= fabsf(ls) ? ls - (hi - m) : m - (hi - ls)};
}

template <int N>
__device__ __forceinline__ void add_values(Stats& a, const float (&x)[N], float mx) {
  if (!(mx <= a.m)) rescale(a, __builtin_elementwise_maximum(a.m, mx));
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = x[e] - a.m;
    const float p = fast_exp(d);
    a.s += p;
    a.u += p * fmaxf(d, kFarBelow);
  }
}

// One wave-wide reduction by lane moves inside rows of 16 and between them; the
// result is in lane 63 and returned to all.  `id` stands in for absent lanes.
template <typename T, typename Op>
__device__ __forceinline__ T wave_reduce(T v, T id, Op op) {
  auto move = [&](auto ctrl, auto rows) {
    const int m = __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, id), __builtin_bit_cast(int, v),
                                              decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v = op(v, __builtin_bit_cast(T, m));
  };
  using I = std::integral_constant<int, 0xf>;
  move(std::integral_constant<int, 0x111>{}, I{});       // from 1, 2, 4, 8 lanes below in the row
  move(std::integral_constant<int, 0x112>{}, I{});
  move(std::integral_constant<int, 0x114>{}, I{});
  move(std::integral_constant<int, 0x118>{}, I{});
  move(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});   // row ends to the next row
  move(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});   // lane 31 to the upper half
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

__device__ __forceinline__ Stats wave_join(Stats a) {
  const float M = wave_reduce(a.m, kLowest, [](float p, float q) { return __builtin_elementwise_maximum(p, q); });
  rescale(a, M);
  auto add = [](float p, float q) { return p + q; };
  return {M, wave_reduce(a.s, 0.f, add), wave_reduce(a.u, 0.f, add)};
}

// ---------------------------------------------------------------------------
// The largest logits.  Lane j < k of a wave holds the j-th best (key, index).
// Keys order floats as unsigned integers: -0 equals +0, NaN above everything,
// 0 is no entry; equal keys order by the lower index.
// ---------------------------------------------------------------------------
__device__ __forceinline__ unsigned key_of(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  const unsigned b = (key & 0x80000000u) ? (key & 0x7fffffffu) : ~key;
  return __builtin_bit_cast(float, b);      // the NaN key maps to a NaN
}

struct Top {
  unsigned key;
  int idx;
  unsigned kth;      // the k-th best's key and index, the same in every lane
  int kth_idx;
  float thr;         // its value; a new x with x <= thr cannot enter
};

__device__ __forceinline__ bool before(unsigned ka, int ia, unsigned kb, int ib) {
  return ka > kb || (ka == kb && ia < ib);
}

__device__ __forceinline__ void top_clear(Top& t) {
  t.key = t.kth = 0;
  t.idx = t.kth_idx = 0x7fffffff;
  t.thr = -__builtin_inff();
}

// the value of the lane below, `first` in lane 0
__device__ __forceinline__ int from_below(int v, int first) {
  return __builtin_amdgcn_update_dpp(first, v, 0x138, 0xf, 0xf, false);
}

__device__ __forceinline__ void top_insert(Top& t, int k, unsigned key, int idx) {
  const unsigned pk = static_cast<unsigned>(from_below(static_cast<int>(t.key), -1));
  const int pi = from_below(t.idx, -1);                        // lane 0: before every entry
  const bool here = !before(t.key, t.idx, key, idx), prev = !before(pk, pi, key, idx);
  t.key = here ? (prev ? pk : key) : t.key;                    // lanes from k on hold what fell out
  t.idx = here ? (prev ? pi : idx) : t.idx;
  t.kth = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(t.key), k - 1));
  t.kth_idx = __builtin_amdgcn_readlane(t.idx, k - 1);
  t.thr = t.kth == 0 ? -__builtin_inff() : value_of(t.kth);
}

// Put what belongs there of G stretches of 8 values a lane (key 0: none; `first`
// is the lane's first index, stretches are `step` apart): the wave's best
// remaining one at a time, so that at most k insertions follow whatever the
// order.  Of equal keys the lowest stretch, lane and value is the lowest index.
// A step is one reduction over the wave and moves between neighbouring lanes, no
// trip through LDS; what it costs is its chain of some 80 dependent instructions,
// so 4 stretches share the steps: 8 rows of 32768 bf16 logits take 4.8 us without
// alternatives and 13.3 us with 5 (24 us with shuffles through LDS and a stretch at
// a time, 17 us with lane moves and a stretch at a time).
template <int G>
__device__ __forceinline__ void top_offer(Top& t, int k, unsigned (&key)[G][8], int first, int step) {
  auto larger = [](unsigned p, unsigned q) { return max(p, q); };
  unsigned best[G];
  auto rate = [&](int q) {
    best[q] = key[q][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) best[q] = max(best[q], key[q][e]);
  };
#pragma unroll
  for (int q = 0; q < G; ++q) rate(q);
  while (true) {
    unsigned mine = best[0];
#pragma unroll
    for (int q = 1; q < G; ++q) mine = max(mine, best[q]);
    const unsigned bk = wave_reduce(mine, 0u, larger);
    if (bk == 0 || bk < t.kth) return;
    unsigned long long at = 0;
    int from = 0;
#pragma unroll
    for (int q = G - 1; q >= 0; --q) {
      const unsigned long long in = __ballot(best[q] == bk);
      at = in != 0 ? in : at;
      from = in != 0 ? q : from;
    }
    const int lane = __ffsll(at) - 1;
    const bool taken = static_cast<int>(threadIdx.x & 63) == lane;
    int own = 0;
#pragma unroll
    for (int q = 0; q < G; ++q) {
      if (q != from) continue;
#pragma unroll
      for (int e = 7; e >= 0; --e) own = key[q][e] == bk ? e : own;
    }
    const int bi = __builtin_amdgcn_readlane(first + own, lane) + from * step;
    if (!before(bk, bi, t.kth, t.kth_idx)) return;
    top_insert(t, k, bk, bi);
    const int gone = taken ? own : -1;
#pragma unroll
    for (int q = 0; q < G; ++q) {
      if (q != from) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) key[q][e] = e == gone ? 0u : key[q][e];
      rate(q);
    }
  }
}

// The same for N (key, index) pairs a lane in any order
template <int N>
__device__ __forceinline__ void top_join(Top& t, int k, unsigned (&key)[N], const int (&idx)[N]) {
  auto larger = [](unsigned p, unsigned q) { return max(p, q); };
  while (true) {
    unsigned mine = key[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mine = max(mine, key[e]);
    const unsigned bk = wave_reduce(mine, 0u, larger);
    if (bk == 0 || bk < t.kth) return;
    int own = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < N; ++e) own = key[e] == bk ? min(own, idx[e]) : own;
    unsigned long long at = __ballot(mine == bk);
    if ((at & (at - 1)) != 0) {                                // equal keys in several lanes
      const unsigned low = wave_reduce(mine == bk ? ~static_cast<unsigned>(own) : 0u, 0u, larger);
      at = __ballot(mine == bk && ~static_cast<unsigned>(own) == low);
    }
    const int bi = __builtin_amdgcn_readlane(own, __ffsll(at) - 1);
    if (!before(bk, bi, t.kth, t.kth_idx)) return;
    top_insert(t, k, bk, bi);
#pragma unroll
    for (int e = 0; e < N; ++e) key[e] = idx[e] == bi ? 0u : key[e];
  }
}

// ---------------------------------------------------------------------------
// Walk a row in index order: f(x[8], first index, valid) per lane, wave w of nw
// taking every nw-th stretch of 512.  16-byte loads from the first aligned
// element on; the few elements before it and after the last whole stretch go one
// by one through the same call.
// ---------------------------------------------------------------------------
constexpr int kPer = 8;
constexpr int kStretch = 64 * kPer;

// 8 logits as they came, untouched until values takes them out
template <typename T>
struct Raw {
  u32x4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p) {
  Raw<T> r;
#pragma unroll
  for (int b = 0; b < static_cast<int>(sizeof(T) / 2); ++b) r.v[b] = reinterpret_cast<const u32x4*>(p)[b];
  return r;
}

template <typename T>
__device__ __forceinline__ void values(const Raw<T>& r, float (&x)[kPer]) {
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if constexpr (sizeof(T) == 4) {
      const unsigned word = r.v[e / 4][e % 4];       // a bit cast of the element itself takes the vector's first
      x[e] = __builtin_bit_cast(float, word);
    } else
      x[e] = to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(r.v[0][e / 2] >> (e % 2 * 16))));
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[kPer]) {
  if constexpr (sizeof(T) == 4) {
    f32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = x[e];
      b[e] = x[4 + e];
    }
    reinterpret_cast<f32x4*>(p)[0] = a;
    reinterpret_cast<f32x4*>(p)[1] = b;
  } else {
    union {
      u32x4 v;
      T t[kPer];
    } q;
#pragma unroll
    for (int e = 0; e < kPer; ++e) q.t[e] = from_f32<T>(x[e]);
    *reinterpret_cast<u32x4*>(p) = q.v;
  }
}

// elements before the first 16-byte aligned one
template <typename T>
__device__ __forceinline__ int head_of(const T* row, int64_t n) {
  const int h = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
  return static_cast<int>(min(static_cast<int64_t>(h), n));
}

// Stretches of 512 of a row, after the few elements before its first aligned one
struct Span {
  int head, body;          // first aligned index, whole stretches
};

template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int n) {
  const int h = head_of(row, n);
  return {h, (n - h) / kStretch};
}

// the elements before the first and behind the last whole stretch
template <typename T, typename F>
__device__ __forceinline__ void walk_head(const T* row, const Span& sp, int w, F&& f) {
  if (w != 0 || sp.head == 0) return;            // at most 7, one a lane
  const int lane = threadIdx.x & 63;
  const bool in = lane < sp.head;
  float x[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = -__builtin_inff();
  if (in) x[0] = to_f32(row[lane]);
  f(x, lane, in ? 1 : 0);
}

template <typename T, typename F>
__device__ __forceinline__ void walk_tail(const T* row, int n, const Span& sp, int w, int nw, F&& f) {
  const int t0 = sp.head + sp.body * kStretch;
  if (t0 >= n || sp.body % nw != w) return;
  const int i = t0 + (threadIdx.x & 63) * kPer;
  const int valid = max(0, min(kPer, n - i));
  float x[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = e < valid ? to_f32(row[i + e]) : -__builtin_inff();
  f(x, i, valid);
}

// The whole row, G stretches of a wave at a time: f(x[G][8], first index, step
// between stretches, valid).  The next ones' loads are in flight behind the work:
// 4096 rows of 131072 bf16 logits 195-200 us (5.4 TB/s), 203 us with one at a time.
template <int G, typename T, typename F>
__device__ __forceinline__ void walk(const T* row, int n, int w, int nw, F&& f) {
  const int lane = threadIdx.x & 63;
  const Span sp = span_of(row, n);
  auto one = [&](float (&x)[kPer], int i, int valid) {
    float v[1][kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[0][e] = x[e];
    f(v, i, 0, valid);
  };
  walk_head(row, sp, w, one);
  const int step = nw * kStretch;
  const T* const body = row + sp.head + lane * kPer;
  Raw<T> cur[G], nxt[G];
  auto fetch = [&](Raw<T>(&r)[G], int b) {
#pragma unroll
    for (int q = 0; q < G; ++q)
      if (b + q * nw < sp.body) r[q] = load8(body + (b + q * nw) * kStretch);
  };
  fetch(cur, w);
  for (int b = w; b < sp.body; b += G * nw) {
    const int i = sp.head + b * kStretch + lane * kPer;
    fetch(nxt, b + G * nw);
    if (b + (G - 1) * nw < sp.body) {
      float x[G][kPer];
#pragma unroll
      for (int q = 0; q < G; ++q) values(cur[q], x[q]);
      f(x, i, step, kPer);
    } else {
#pragma unroll
      for (int q = 0; q < G - 1; ++q)
        if (b + q * nw < sp.body) {
          float x[1][kPer];
          values(cur[q], x[0]);
          f(x, i + q * step, 0, kPer);
        }
    }
#pragma unroll
    for (int q = 0; q < G; ++q) cur[q] = nxt[q];
  }
  walk_tail(row, n, sp, w, nw, one);
}

struct Args {
  int64_t ldl;
  const int64_t* targets;
  int64_t rows;
  int vocab;
  int64_t ignore;
  int top;
  float* logp;
  float* entropy;
  float* lse;
  float* lse_rest;
  float* top_logp;
  int64_t* top_ids;
  const float* grad_logp;
  const float* grad_entropy;
  int64_t ldg;
};

// the gradient of 8 logits of a row, given its lse and entropy
template <typename T>
struct RowGrad {
  T* grow;
  int64_t target;
  Lse lse;
  float ent, gl, ge;
  bool same;                // logits and gradient are aligned alike

  __device__ __forceinline__ void operator()(float (&x)[kPer], int i, int valid) const {
    float g[kPer] = {};
    // nothing of a row that is left out, whatever it holds: 0 * p would be NaN with p
    if (gl != 0.f || ge != 0.f) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float l = lse.below(x[e]);
        const float p = fast_exp(l);
        float v = -gl * p;
        if (ge != 0.f) v -= ge * p * (fmaxf(l, kFarBelow) + ent);
        if (i + e == target) v += gl;
        g[e] = v;
      }
    }
    if (valid == kPer && same) {
      store8(grow + i, g);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (e < valid) grow[i + e] = from_f32<T>(g[e]);
    }
  }
};

// A 16-bit gradient leaves the rest out where |lse| < 16: it moves p by less than
// 2^-21 of itself (8 roundings of a float; the sums may have left as much), and the
// gradient from lse alone then has the same bits.
template <typename T>
__device__ __forceinline__ RowGrad<T> row_grad(const T* row, T* grow, int64_t target, Lse lse, float ent, float gl,
                                               float ge) {
  if (sizeof(T) == 2 && fabsf(lse.hi) < 16.f) lse.lo = 0.f;
  return {grow, target, lse, ent, gl, ge,
          ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0};
}

constexpr int kAhead = 4;                 // stretches a wave takes at a time

// WAVES waves a row, 4 waves (or WAVES, if more) a workgroup.  KEEP > 0: a wave
// holds its up to KEEP stretches in registers from the one read to the gradient.
// Bound by memory: 4096 rows of 50001 bf16 logits and their gradient 193 us (4.2
// TB/s read and written; rows start at odd places), 249 us read twice; 189 us where a
// tenth of the rows is ignored.  65536 wide 229 us (4.7 TB/s); 128256, read twice,
// 640 us (4.9 TB/s of three passes; two would be 409 us at a copy's rate).
template <typename T, int WAVES, bool TOP, bool GRAD, int KEEP>
__global__ void __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64)
    logprob_kernel(const T* logits, Args a, T* grad) {
  static_assert(WAVES == 1 || WAVES >= 4, "a workgroup's waves share the barrier of one row");
  constexpr int kRows = WAVES < 4 ? 4 / WAVES : 1;
  __shared__ Stats sh_stats[kRows * WAVES];
  __shared__ unsigned sh_key[TOP ? kRows * WAVES * SRA_TOKEN_MAX_TOP : 1];
  __shared__ int sh_idx[TOP ? kRows * WAVES * SRA_TOKEN_MAX_TOP : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int local = wave / WAVES, w = wave % WAVES;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + local;
  const bool live = r < a.rows;

  Stats st{kLowest, 0.f, 0.f};
  Top t;
  top_clear(t);
  const T* row = logits + (live ? r : 0) * a.ldl;
  auto take_all = [&](auto& x, int i, int step, int valid) {
    constexpr int G = sizeof(x) / sizeof(x[0]);
    float all = -__builtin_inff();
#pragma unroll
    for (int q = 0; q < G; ++q) {
      float mx = x[q][0];
#pragma unroll
      for (int e = 1; e < kPer; ++e) mx = __builtin_elementwise_maximum(mx, x[q][e]);
      add_values(st, x[q], mx);
      all = __builtin_elementwise_maximum(all, mx);
    }
    if constexpr (TOP) {
      if (__ballot(t.kth == 0 || !(all <= t.thr)) != 0) {
        unsigned key[G][kPer];
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
          for (int e = 0; e < kPer; ++e) key[q][e] = e < valid ? key_of(x[q][e]) : 0u;
        top_offer(t, a.top, key, i, step);
      }
    }
  };
  auto take = [&](float (&x)[kPer], int i, int valid) {
    float v[1][kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[0][e] = x[e];
    take_all(v, i, 0, valid);
  };
  Raw<T> kept[KEEP > 0 ? KEEP : 1];
  const Span sp = span_of(row, a.vocab);
  if (live) {
    if constexpr (KEEP > 0) {
#pragma unroll
      for (int q = 0; q < KEEP; ++q)
        if (w + q * WAVES < sp.body) kept[q] = load8(row + sp.head + (w + q * WAVES) * kStretch + lane * kPer);
      walk_head(row, sp, w, take);
#pragma unroll
      for (int q = 0; q < KEEP; ++q)
        if (w + q * WAVES < sp.body) {
          float x[kPer];
          values(kept[q], x);
          take(x, sp.head + (w + q * WAVES) * kStretch + lane * kPer, kPer);
        }
      walk_tail(row, a.vocab, sp, w, WAVES, take);
    } else {
      walk<kAhead>(row, a.vocab, w, WAVES, take_all);
    }
  }
  st = wave_join(st);
  if constexpr (WAVES > 1) {
    if (lane == 0) sh_stats[wave] = st;
    if constexpr (TOP) {
      if (lane < a.top) {
        sh_key[wave * SRA_TOKEN_MAX_TOP + lane] = t.key;
        sh_idx[wave * SRA_TOKEN_MAX_TOP + lane] = t.idx;
      }
    }
    __syncthreads();
    // every wave joins them in the same order
    st = sh_stats[0];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) join(st, sh_stats[q]);
    if constexpr (TOP) {
      if (w == 0) {
        // all lists at once: entry e of a lane is number e * 64 + lane
        constexpr int kAll = WAVES * SRA_TOKEN_MAX_TOP / 64;
        unsigned key[kAll];
        int idx[kAll];
#pragma unroll
        for (int e = 0; e < kAll; ++e) {
          const int q = e * 64 + lane, from = q / a.top * SRA_TOKEN_MAX_TOP + q % a.top;
          const bool in = q < WAVES * a.top;
          key[e] = in ? sh_key[from] : 0u;
          idx[e] = in ? sh_idx[from] : 0x7fffffff;
        }
        top_clear(t);
        top_join(t, a.top, key, idx);
      }
    }
  }
  if (!live) return;
  const float ls = logf(st.s);
  const Lse lse = lse_of(st.m, ls);
  const float ent = ls - st.u / st.s;
  const int64_t target = a.targets[r];
  const bool ignored = target == a.ignore;
  const bool bad = !ignored && (target < 0 || target >= a.vocab);
  if (w == 0 && lane == 0) {
    float lp = 0.f;
    if (bad) {
      count_row_fault();
      lp = __builtin_nanf("");
    } else if (!ignored) {
      lp = lse.below(to_f32(row[target]));
    }
    a.logp[r] = lp;
    a.lse[r] = lse.hi;
    if (a.lse_rest != nullptr) a.lse_rest[r] = lse.lo;
    if (a.entropy != nullptr) a.entropy[r] = ent;
  }
  if constexpr (TOP) {
    if (w == 0 && lane < a.top) {
      a.top_logp[r * a.top + lane] = lse.below(value_of(t.key));
      a.top_ids[r * a.top + lane] = t.idx;
    }
  }
  if constexpr (GRAD) {
    // the target is read before an in-place gradient replaces it
    if constexpr (WAVES > 1) __syncthreads(); else __threadfence_block();
    const bool none = ignored || bad;
    const auto put = row_grad(row, grad + r * a.ldg, none ? -1 : target, lse, ent, none ? 0.f : a.grad_logp[r],
                              a.grad_entropy != nullptr ? a.grad_entropy[r] : 0.f);
    if constexpr (KEEP > 0) {
      walk_head(row, sp, w, put);
#pragma unroll
      for (int q = 0; q < KEEP; ++q)
        if (w + q * WAVES < sp.body) {
          float x[kPer];
          values(kept[q], x);
          put(x, sp.head + (w + q * WAVES) * kStretch + lane * kPer, kPer);
        }
      walk_tail(row, a.vocab, sp, w, WAVES, put);
    } else {
      walk<1>(row, a.vocab, w, WAVES, [&](float (&x)[1][kPer], int i, int, int valid) { put(x[0], i, valid); });
    }
  }
}

// the gradient from a forward pass's lse and entropy: 4 waves take a stretch of
// 8192 of a row (4096 rows of bf16 logits: 50001 wide 179 us, 4.6 TB/s; 128256 425
// us, 4.9 TB/s)
constexpr int kGradSpan = 8192;

template <typename T>
__global__ void __launch_bounds__(256) logprob_grad_kernel(const T* logits, Args a, const float* __restrict__ lse,
                                                           const float* __restrict__ lse_rest,
                                                           const float* __restrict__ entropy, T* grad) {
  const int64_t r = blockIdx.x;
  const int from = blockIdx.y * kGradSpan;
  const int n = min(kGradSpan, a.vocab - from);
  int64_t target = a.targets[r];
  float gl = a.grad_logp[r];
  const bool ignored = target == a.ignore;
  if (ignored || target < 0 || target >= a.vocab) {
    if (!ignored && from == 0 && threadIdx.x == 0) count_row_fault();
    gl = 0.f;
    target = -1;
  }
  const float ge = a.grad_entropy != nullptr ? a.grad_entropy[r] : 0.f;
  const float ent = a.grad_entropy != nullptr ? entropy[r] : 0.f;
  const T* row = logits + r * a.ldl + from;
  const Lse both{lse[r], lse_rest != nullptr ? lse_rest[r] : 0.f};
  const auto put = row_grad(row, grad + r * a.ldg + from, target - from, both, ent, gl, ge);
  walk<1>(row, n, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), 4,
          [&](float (&x)[1][kPer], int i, int, int valid) { put(x[0], i, valid); });
}

static int check_logits(const void* logits, int64_t ldl, int32_t dtype, const int64_t* targets, int64_t rows,
                        int64_t vocab) {
  if (int rc = check_dtype(dtype, "dtype")) return rc;
  SRA_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), SRA_ERR_SHAPE, "rows must be in [0, 2^31), got %lld",
              static_cast<long long>(rows));
  SRA_REQUIRE(vocab >= 1 && vocab < (int64_t{1} << 28), SRA_ERR_SHAPE, "vocab must be in [1, 2^28), got %lld",
              static_cast<long long>(vocab));
  SRA_REQUIRE(rows == 0 || (logits != nullptr && targets != nullptr), SRA_ERR_ARG,
              "logits and targets must be non-null");
  SRA_REQUIRE(rows <= 1 || ldl >= vocab, SRA_ERR_SHAPE, "logits need a row stride >= %lld, got %lld",
              static_cast<long long>(vocab), static_cast<long long>(ldl));
  SRA_REQUIRE((reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype)) == 0, SRA_ERR_ARG,
              "logits are not aligned to their type");
  return SRA_OK;
}

static int check_grad(const void* logits, int64_t ldl, const void* grad, int64_t ldg, int64_t rows, int64_t vocab,
                      int32_t dtype) {
  SRA_REQUIRE(rows <= 1 || ldg >= vocab, SRA_ERR_SHAPE, "grad needs a row stride >= %lld, got %lld",
              static_cast<long long>(vocab), static_cast<long long>(ldg));
  SRA_REQUIRE(grad != logits || ldg == ldl || rows <= 1, SRA_ERR_SHAPE,
              "logits and grad are one buffer with two row strides");
  SRA_REQUIRE((reinterpret_cast<uintptr_t>(grad) % dtype_size(dtype)) == 0, SRA_ERR_ARG,
              "grad is not aligned to its type");
  return SRA_OK;
}

template <typename T, int WAVES, int KEEP>
static int launch_rows(const void* logits, const Args& a, void* grad, hipStream_t st) {
  constexpr int kRows = WAVES < 4 ? 4 / WAVES : 1;
  const dim3 grid(static_cast<unsigned>(cdiv(a.rows, kRows))), block(WAVES < 4 ? 256 : WAVES * 64);
  if (int rc = check_launch(grid.x, static_cast<int>(block.x))) return rc;
  const T* l = static_cast<const T*>(logits);
  T* g = static_cast<T*>(grad);
  if (g != nullptr) {
    if (a.top > 0)
      hipLaunchKernelGGL((logprob_kernel<T, WAVES, true, true, KEEP>), grid, block, 0, st, l, a, g);
    else
      hipLaunchKernelGGL((logprob_kernel<T, WAVES, false, true, KEEP>), grid, block, 0, st, l, a, g);
  } else if constexpr (KEEP == 0) {
    if (a.top > 0)
      hipLaunchKernelGGL((logprob_kernel<T, WAVES, true, false, 0>), grid, block, 0, st, l, a, g);
    else
      hipLaunchKernelGGL((logprob_kernel<T, WAVES, false, false, 0>), grid, block, 0, st, l, a, g);
  }
  return launch_status("logprob_kernel");
}

// Waves a row: one for rows of up to 2048 logits (4096 rows of 1024 5.2 us, 7.0 us
// with 4 waves; 8 rows of 4096 6.3 us, 4.3 us with 16); 4 where the rows fill the
// card, 16 where they do not (rows of 32768: 256 8.6 us with 4, 7.7 with 16; 512
// 12.4, 13.9; 2048 34.7, 44.5).  With the gradient, 8 waves keep a row of up to
// 65536 16-bit (32768 float32) logits in registers, a quarter of them for rows a
// quarter as long; longer rows are read twice.  4 waves with twice the registers
// put three rows of 16-bit logits on a compute unit instead of two, where there are
// that many (bf16, 32000 wide: 512 rows 25.6 us with 8, 27.7 with 4; 768 35.6, 33.4;
// 4096 160, 141; 4096 of 5000 37.4, 29.9; float32 gains nothing).
template <typename T>
static int launch(const void* logits, const Args& a, void* grad, hipStream_t st) {
  constexpr int kMost = sizeof(T) == 4 ? 8 : 16;
  if (a.vocab <= 2048) return launch_rows<T, 1, 0>(logits, a, grad, st);
  if (grad != nullptr && a.vocab <= 8 * kMost * kStretch) {
    const bool quarter = a.vocab <= 8 * kMost / 4 * kStretch;
    if constexpr (sizeof(T) == 2)
      if (a.rows >= 768)
        return quarter ? launch_rows<T, 4, kMost / 2>(logits, a, grad, st)
                       : launch_rows<T, 4, 2 * kMost>(logits, a, grad, st);
    return quarter ? launch_rows<T, 8, kMost / 4>(logits, a, grad, st) : launch_rows<T, 8, kMost>(logits, a, grad, st);
  }
  return a.rows < 512 ? launch_rows<T, 16, 0>(logits, a, grad, st) : launch_rows<T, 4, 0>(logits, a, grad, st);
}

template <typename F>
static int with_type(int32_t dtype, F&& f) {
  if (dtype == SRA_F32) return f(float{});
  if (dtype == SRA_BF16) return f(__bf16{});
  return f(_Float16{});
}

}  // namespace sra

using namespace sra;

extern "C" int sra_token_logprobs_split(const void* logits, int64_t ldl, int32_t dtype, const int64_t* targets,
                                        int64_t rows, int64_t vocab, int64_t ignore, int32_t top, float* logp,
                                        float* entropy, float* lse, float* lse_rest, float* top_logp,
                                        int64_t* top_ids, const float* grad_logp, const float* grad_entropy,
                                        void* grad, int64_t ldg, void* stream) {
  if (int rc = check_logits(logits, ldl, dtype, targets, rows, vocab)) return rc;
  SRA_REQUIRE(top >= 0 && top <= vocab, SRA_ERR_ARG, "top must be in [0, vocab], got %d", top);
  SRA_REQUIRE(top <= SRA_TOKEN_MAX_TOP, SRA_ERR_UNSUPPORTED, "top %d is above %d", top, SRA_TOKEN_MAX_TOP);
  SRA_REQUIRE(rows == 0 || (logp != nullptr && lse != nullptr), SRA_ERR_ARG, "logp and lse must be non-null");
  SRA_REQUIRE(rows == 0 || top == 0 || (top_logp != nullptr && top_ids != nullptr), SRA_ERR_ARG,
              "top_logp and top_ids must be non-null");
  SRA_REQUIRE(grad == nullptr || grad_logp != nullptr, SRA_ERR_ARG, "the gradient needs grad_logp");
  if (grad != nullptr)
    if (int rc = check_grad(logits, ldl, grad, ldg, rows, vocab, dtype)) return rc;
  if (rows == 0) return SRA_OK;
  const Args a{ldl, targets, rows, static_cast<int>(vocab), ignore, top, logp, entropy, lse, lse_rest, top_logp,
               top_ids, grad_logp, grad_entropy, ldg};
  return with_type(dtype, [&](auto t) {
    return launch<decltype(t)>(logits, a, grad, static_cast<hipStream_t>(stream));
  });
}

extern "C" int sra_token_logprobs(const void* logits, int64_t ldl, int32_t dtype, const int64_t* targets,
                                  int64_t rows, int64_t vocab, int64_t ignore, int32_t top, float* logp,
                                  float* entropy, float* lse, float* top_logp, int64_t* top_ids,
                                  const float* grad_logp, const float* grad_entropy, void* grad, int64_t ldg,
                                  void* stream) {
  return sra_token_logprobs_split(logits, ldl, dtype, targets, rows, vocab, ignore, top, logp, entropy, lse, nullptr,
                                  top_logp, top_ids, grad_logp, grad_entropy, grad, ldg, stream);
}

extern "C" int sra_token_logprobs_grad_split(const void* logits, int64_t ldl, int32_t dtype, const int64_t* targets,
                                             int64_t rows, int64_t vocab, int64_t ignore, const float* lse,
                                             const float* lse_rest, const float* entropy, const float* grad_logp,
                                             const float* grad_entropy, void* grad, int64_t ldg, void* stream) {
  if (int rc = check_logits(logits, ldl, dtype, targets, rows, vocab)) return rc;
  if (rows == 0) return SRA_OK;
  SRA_REQUIRE(lse != nullptr && grad_logp != nullptr && grad != nullptr, SRA_ERR_ARG,
              "lse, grad_logp and grad must be non-null");
  SRA_REQUIRE(grad_entropy == nullptr || entropy != nullptr, SRA_ERR_ARG,
              "grad_entropy needs the forward pass's entropy");
  if (int rc = check_grad(logits, ldl, grad, ldg, rows, vocab, dtype)) return rc;
  const Args a{ldl, targets, rows, static_cast<int>(vocab), ignore, 0, nullptr, nullptr, nullptr, nullptr, nullptr,
               nullptr, grad_logp, grad_entropy, ldg};
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(cdiv(vocab, kGradSpan)));
    if (int rc = check_launch(rows, 256)) return rc;
    hipLaunchKernelGGL((logprob_grad_kernel<T>), grid, dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T*>(logits), a, lse, lse_rest, entropy, static_cast<T*>(grad));
    return launch_status("logprob_grad_kernel");
  });
}

extern "C" int sra_token_logprobs_grad(const void* logits, int64_t ldl, int32_t dtype, const int64_t* targets,
                                       int64_t rows, int64_t vocab, int64_t ignore, const float* lse,
                                       const float* entropy, const float* grad_logp, const float* grad_entropy,
                                       void* grad, int64_t ldg, void* stream) {
  return sra_token_logprobs_grad_split(logits, ldl, dtype, targets, rows, vocab, ignore, lse, nullptr, entropy,
                                       grad_logp, grad_entropy, grad, ldg, stream);
}

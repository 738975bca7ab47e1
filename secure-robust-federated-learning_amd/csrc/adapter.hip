// k12 — low-rank adapters of many clients beside a shared projection.
//
//   h_t = A_c x_t,  out_t = base_t + scale * B_c h_t          (c = slot of t)
//   z_t = B_c' dout_t,  dx_t = dxbase_t + scale * A_c' z_t
//   dA_c = scale * sum_t z_t x_t',  dB_c = scale * sum_t dout_t h_t'
//
// Three products on the matrix units, all bound by memory: shrink (x to the
// rank), expand (the rank to a row, added to base) and outer (a sum over the
// tokens of a client).  The backward pass is the same three with A and B
// exchanged, so shrink and expand take a weight stored either way round.
//
// Arithmetic.  Sums are float32.  16-bit activations run on the bf16 units
// (v_mfma_f32_16x16x32_bf16): a bf16 value is one term, an fp16 one two (the
// nearest bf16 and the rest), a float32 one (weights, h, z) three, which hold all
// its 24 bits, where the result stays float32 (h, z, the gradients of A and B),
// and two where it is rounded to 16 bits anyway (out, dx).  Products of terms
// below 2^-16 (or 2^-8) of the whole are left out.  Memory bounds all three
// products, so the matrix instructions, up to five for one, have room.  A product
// with an infinity is then the sum of several that may have opposite signs: it
// comes out infinite or NaN.  A finite one keeps its digits up to float32's largest
// value, but sums within 2^-8 of that may pass it on their way.  float32
// activations run on the float32 units (v_mfma_f32_16x16x4_f32).
//
// Layout.  A lane (n = lane % 16, g = lane / 16) of a 16x16 product holds row or
// column n of its operands with the inner indices g * 8 .. g * 8 + 7 and, of the
// result, column n of rows g * 4 .. g * 4 + 3.  Both operands may permute rows
// and inner indices alike, which the kernels use to make 8 consecutive values of
// memory one lane's load or store.
#include <algorithm>
#include <type_traits>

#include "lm_common.hpp"

namespace sra {

unsigned int adapter_row_faults(bool reset) { return tu_row_faults(reset); }

// ---------------------------------------------------------------------------
// 8 values a lane, and their products
// ---------------------------------------------------------------------------
// Two values in a word, rounded to nearest even, and back
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, pair));
}
template <typename T>
__device__ __forceinline__ f32x2 unpack2(unsigned w) {
  if constexpr (std::is_same_v<T, __bf16>)
    return f32x2{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
  else
    return f32x2{to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(w))),
                 to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(w >> 16)))};
}

// N stored values as they came, in words: a load's registers stay untouched, and
// unwaited for, until get takes a value out of them.
template <typename S, int N>
struct RawN {
  static constexpr int kWords = N * static_cast<int>(sizeof(S)) / 4;
  unsigned w[kWords];
  __device__ __forceinline__ S get(int e) const {
    if constexpr (sizeof(S) == 4) {
      const unsigned v = w[e];
      return __builtin_bit_cast(S, v);
    } else {
      return __builtin_bit_cast(S, static_cast<unsigned short>(w[e / 2] >> (e % 2 * 16)));
    }
  }
  // values e and e + 1, e even
  __device__ __forceinline__ f32x2 get2(int e) const {
    if constexpr (sizeof(S) == 4) return f32x2{get(e), get(e + 1)};
    else return unpack2<S>(w[e / 2]);
  }
  __device__ __forceinline__ void set2(int e, float a, float b) {
    if constexpr (sizeof(S) == 4) {
      w[e] = __builtin_bit_cast(unsigned, a);
      w[e + 1] = __builtin_bit_cast(unsigned, b);
    } else {
      w[e / 2] = pack2<S>(a, b);
    }
  }
};
template <typename S>
using Raw8 = RawN<S, 8>;
template <typename S>
using Raw4 = RawN<S, 4>;

// N consecutive elements at any alignment of their type (the hardware's global
// loads take it), in loads of 16 bytes, or one of 8
typedef u32x4 __attribute__((aligned(2))) any_u32x4;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 __attribute__((aligned(2))) any_u32x2;

template <typename S, int N>
__device__ __forceinline__ RawN<S, N> load_n(const S* p) {
  RawN<S, N> r;
  if constexpr (sizeof(r) == 8) {
    const u32x2 v = *reinterpret_cast<const any_u32x2*>(p);
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
#pragma unroll
    for (int b = 0; b < r.kWords / 4; ++b) {
      const u32x4 v = reinterpret_cast<const any_u32x4*>(p)[b];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[b * 4 + e] = v[e];
    }
  }
  return r;
}

// Elements o .. o + N - 1 of n >= N that lie one behind the other, where those
// that do not matter may be others: the last N of all where o + N is beyond the
// end, to be moved into place by settle when they are used.  So every lane's load
// is one without a branch, and many are in flight at once.
template <typename S, int N>
__device__ __forceinline__ RawN<S, N> load_at(const S* p, int64_t o, int64_t n) {
  return load_n<S, N>(p + min(o, n - N));
}

template <typename S, int N>
__device__ __forceinline__ void settle(RawN<S, N>& r, int64_t o, int64_t n) {
  const int64_t d = o - (n - N);
  if (__ballot(d > 0 && d < N) == 0) return;
  const int by = d > 0 ? static_cast<int>(d) : 0;
  constexpr int kWords = RawN<S, N>::kWords, kPer = 4 / sizeof(S);
  // by constants and masks: registers have no address to choose by
  auto words_down = [&](auto step) {
    constexpr int kStep = decltype(step)::value;
    if constexpr (kStep < kWords) {
      const unsigned on = (by & (kStep * kPer)) != 0 ? 0xffffffffu : 0u;
#pragma unroll
      for (int e = 0; e + kStep < kWords; ++e) r.w[e] = (r.w[e + kStep] & on) | (r.w[e] & ~on);
    }
  };
  words_down(std::integral_constant<int, 4>{});
  words_down(std::integral_constant<int, 2>{});
  words_down(std::integral_constant<int, 1>{});
  if constexpr (sizeof(S) == 2) {
    const unsigned on = (by & 1) != 0 ? 0xffffffffu : 0u;
#pragma unroll
    for (int e = 0; e < kWords; ++e) {
      const unsigned next = e + 1 < kWords ? r.w[e + 1] : 0u;
      r.w[e] = ((r.w[e] >> 16 | next << 16) & on) | (r.w[e] & ~on);
    }
  }
}

// values from `valid` on become zero
template <typename S, int N>
__device__ __forceinline__ void cut(RawN<S, N>& r, int valid) {
#pragma unroll
  for (int b = 0; b < RawN<S, N>::kWords; ++b) {
    if constexpr (sizeof(S) == 4) r.w[b] &= b < valid ? 0xffffffffu : 0u;
    else r.w[b] &= 2 * b + 1 < valid ? 0xffffffffu : 2 * b < valid ? 0xffffu : 0u;
  }
}

template <typename S, int N>
__device__ __forceinline__ void store_n(S* p, const RawN<S, N>& r, int valid) {
  if (valid >= N) {
    if constexpr (sizeof(r) == 8) {
      *reinterpret_cast<any_u32x2*>(p) = u32x2{r.w[0], r.w[1]};
    } else {
#pragma unroll
      for (int b = 0; b < r.kWords / 4; ++b)
        reinterpret_cast<any_u32x4*>(p)[b] = u32x4{r.w[b * 4], r.w[b * 4 + 1], r.w[b * 4 + 2], r.w[b * 4 + 3]};
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < valid) p[e] = r.get(e);
  }
}

// 8 operand values a lane: bf16 terms, two values a word, or floats
template <int N>
struct Terms {
  unsigned t[N][4];
  __device__ __forceinline__ bf16x8 term(int i) const {
    return __builtin_bit_cast(bf16x8, u32x4{t[i][0], t[i][1], t[i][2], t[i][3]});
  }
};
struct Floats {
  float v[8];
};

// the operand that T's matrix units take for stored values S
template <typename T, typename S, bool FULL = false>
using Frag = std::conditional_t<std::is_same_v<T, float>, Floats,
                                Terms<std::is_same_v<S, __bf16> ? 1 : std::is_same_v<S, float> && FULL ? 3 : 2>>;

// values e and e + 1, e even, of type S: the nearest bf16, that of the rest, that of
// its rest.  A float32 above bf16's largest value, whose nearest bf16 is infinite,
// has that largest one as its first term.
constexpr float kMostBf16 = 3.3895314e38f;
template <typename S, int N>
__device__ __forceinline__ void put2(Terms<N>& f, int e, f32x2 x) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (std::is_same_v<S, float> && i == 0)
      f.t[i][e / 2] = pack2<__bf16>(__builtin_amdgcn_fmed3f(x[0], -kMostBf16, kMostBf16),
                                    __builtin_amdgcn_fmed3f(x[1], -kMostBf16, kMostBf16));
    else
      f.t[i][e / 2] = pack2<__bf16>(x[0], x[1]);
    if (i + 1 < N) {
      const f32x2 h = unpack2<__bf16>(f.t[i][e / 2]);
      x = f32x2{x[0] - h[0], x[1] - h[1]};
    }
  }
}
template <typename S>
__device__ __forceinline__ void put2(Floats& f, int e, f32x2 x) {
  f.v[e] = x[0];
  f.v[e + 1] = x[1];
}

template <typename F, typename S>
__device__ __forceinline__ F frag_of(const Raw8<S>& r) {
  F f;
  if constexpr (std::is_same_v<S, __bf16>) {
#pragma unroll
    for (int b = 0; b < 4; ++b) f.t[0][b] = r.w[b];
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) put2<S>(f, e, r.get2(e));
  }
  return f;
}

// column a of 8 rows
template <typename F, typename S, int N>
__device__ __forceinline__ F column_of(const RawN<S, N> (&r)[8], int a) {
  F f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    if constexpr (std::is_same_v<S, __bf16>)
      f.t[0][e / 2] = __builtin_amdgcn_perm(r[e + 1].w[a / 2], r[e].w[a / 2], a % 2 ? 0x07060302u : 0x05040100u);
    else
      put2<S>(f, e, f32x2{to_f32(r[e].get(a)), to_f32(r[e + 1].get(a))});
  }
  return f;
}

// A fragment in LDS: its 16-byte pieces in planes of their own
template <int N>
__device__ __forceinline__ void put_frag(u32x4* lds, int plane, int at, const Terms<N>& f) {
#pragma unroll
  for (int p = 0; p < N; ++p) lds[p * plane + at] = u32x4{f.t[p][0], f.t[p][1], f.t[p][2], f.t[p][3]};
}
__device__ __forceinline__ void put_frag(u32x4* lds, int plane, int at, const Floats& f) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = f.v[4 * p + e];
    lds[p * plane + at] = __builtin_bit_cast(u32x4, v);
  }
}
template <int N>
__device__ __forceinline__ void get_frag(Terms<N>& f, const u32x4* lds, int plane, int at) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const u32x4 v = lds[p * plane + at];
#pragma unroll
    for (int b = 0; b < 4; ++b) f.t[p][b] = v[b];
  }
}
__device__ __forceinline__ void get_frag(Floats& f, const u32x4* lds, int plane, int at) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const f32x4 v = __builtin_bit_cast(f32x4, lds[p * plane + at]);
#pragma unroll
    for (int e = 0; e < 4; ++e) f.v[4 * p + e] = v[e];
  }
}
template <typename F>
constexpr int kPlanes = sizeof(F) / 16;

// the products of the terms that add up to at least 2^-8 (FULL: 2^-16) of the whole
template <bool FULL, int N, int M>
__device__ __forceinline__ void mma(f32x4& acc, const Terms<N>& a, const Terms<M>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
#pragma unroll
    for (int j = M - 1; j >= 0; --j)
      if (i + j < (FULL ? 3 : 2)) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.term(i), b.term(j), acc, 0, 0, 0);
}

template <bool FULL>
__device__ __forceinline__ void mma(f32x4& acc, const Floats& a, const Floats& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Token tiles.  Segments are cut into tiles of TT tokens that never cross a
// segment.  Segment i starts at e_i, so its tiles may take the numbers from
// e_i / TT + i on: e_{i+1} / TT + i + 1 is never below the last of them.  A
// workgroup finds its tile on the device by searching those numbers; the rows
// before the first and behind the last segment count as segments without a slot.
// The tokens of a bad slot are counted by the first launch of a call that finds
// them, one workgroup a tile.
// ---------------------------------------------------------------------------
struct Segs {
  const int64_t* offsets;
  const int32_t* slots;
  int nseg, nslots;
  int64_t tokens;
};

struct Tile {
  int t0, n, slot;
};

__device__ __forceinline__ int seg_start(const Segs& sg, int i) {
  if (i == 0) return 0;
  if (i == sg.nseg + 2) return static_cast<int>(sg.tokens);
  return static_cast<int>(min(max(sg.offsets[i - 1], int64_t{0}), sg.tokens));
}

template <int TT>
__device__ __forceinline__ Tile find_tile(const Segs& sg, int tile, bool count_faults) {
  const int lane = threadIdx.x & 63, count = sg.nseg + 2;
  int lo, first, end, slot;
  if (count <= 256) {
    // every start and slot in one round of loads: the search costs one trip to memory
    int st[4], sl[4], hits = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = q * 64 + lane;
      st[q] = i < count ? seg_start(sg, i) : static_cast<int>(sg.tokens);
      sl[q] = i >= 1 && i <= sg.nseg ? sg.slots[i - 1] : -1;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = q * 64 + lane;
      hits += __popcll(__ballot(i < count && st[q] / TT + i <= tile));
    }
    lo = max(hits, 1) - 1;
    first = end = static_cast<int>(sg.tokens);
    slot = -1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (lo >> 6 == q) {
        first = __builtin_amdgcn_readlane(st[q], lo & 63);
        slot = __builtin_amdgcn_readlane(sl[q], lo & 63);
      }
      if ((lo + 1) >> 6 == q) end = __builtin_amdgcn_readlane(st[q], (lo + 1) & 63);
    }
  } else {
    lo = 0;
    for (int len = count; len > 1;) {        // 64 candidates at a time
      const int step = (len + 63) >> 6, i = lane * step;
      const bool at = i < len && seg_start(sg, lo + i) / TT + lo + i <= tile;
      const int skip = (max(__popcll(__ballot(at)), 1) - 1) * step;
      lo += skip;
      len = min(step, len - skip);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    first = seg_start(sg, lo);
    end = seg_start(sg, lo + 1);
    slot = lo >= 1 && lo <= sg.nseg ? sg.slots[lo - 1] : -1;
  }
  // numbers that no tile has end here, and so do offsets that do not ascend
  const int64_t t0 = first + static_cast<int64_t>(tile - first / TT - lo) * TT;
  Tile t;
  t.t0 = static_cast<int>(t0);
  t.n = t0 < first ? 0 : static_cast<int>(max(int64_t{0}, min(end - t0, int64_t{TT})));
  t.slot = slot;
  if (t.n > 0 && (slot < -1 || slot >= sg.nslots)) {
    if (count_faults && threadIdx.x == 0) count_row_fault(t.n);
    t.slot = -1;
  }
  return t;
}

template <int TT>
static int tile_count(const Segs& sg) {
  return static_cast<int>(sg.tokens / TT) + sg.nseg + 2;
}

// ---------------------------------------------------------------------------
// Staging.  A load straight into an operand's lanes would take 16 bytes of 16
// rows at a time: every 16 bytes a cache line of its own.  So operands that more
// than one lane group shares, or whose rows are memory's rows, are read in
// whole lines, brought into fragments once a workgroup, and put into LDS as
// pieces (row, c) of 8 inner values.  Their places let any 8 neighbouring lanes of
// a read (rows n, or n * PERM + a for n = 0..15) and of a write fall into
// different banks: row r at (r % PERM) * kStep + r / PERM, with kStep and the
// distance of pieces padded for that.
//
// TR false: element (row, inner) at src[row * ld + inner].  TR true: at
// src[inner * ld + row]; a thread then loads 4 rows of 8 inner values and turns
// them in registers.  fetch and put are apart so that the next stage's loads are
// in flight behind this one's products.
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;

template <typename T, typename S, int ROWS, int PIECES, bool TR, int PERM, bool FULL>
struct Stage {
  using F = Frag<T, S, FULL>;
  static constexpr int kStep = PERM == 8 ? ROWS / 8 + 1 : PERM == 4 ? ROWS / 4 + 2 : 0;
  static constexpr int kPiece = PERM == 1 ? ROWS + 1 : PERM * kStep + (TR ? 4 : 1);
  static constexpr int kPlane = PIECES * kPiece;
  static constexpr int kBytes = kPlane * kPlanes<F> * 16;
  static constexpr int kUnits = TR ? ROWS / 4 * PIECES : ROWS * PIECES;
  static constexpr int kEach = (kUnits + kThreads - 1) / kThreads;
  RawN<S, TR ? 4 : 8> r[kEach][TR ? 8 : 1];                // a line, or 8 to turn
  int64_t ld, total;
  int rows, inner;

  // `total` elements from src on may be read.  Rows from nrows on hold anything
  // (their products are never stored), inner values from ninner on are zero once
  // they are put.
  __device__ __forceinline__ void fetch(const S* src, int64_t ld_, int nrows, int ninner, int64_t total_) {
    ld = ld_;
    total = total_;
    rows = nrows;
    inner = ninner;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int u = unit(q);
      if constexpr (TR) {
        const int row = u % (ROWS / 4) * 4, k = u / (ROWS / 4) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[q][e] = load_at<S, 4>(src, turn_at(k + e, row), total);
      } else {
        r[q][0] = load_at<S, 8>(src, line_at(u), total);
      }
    }
  }

  // threads beyond the units load the last one again and put nothing
  static __device__ __forceinline__ int unit(int q) {
    return min(q * kThreads + static_cast<int>(threadIdx.x), kUnits - 1);
  }

  static __device__ __forceinline__ int place(int row, int c) {
    return c * kPiece + (PERM == 1 ? row : row % PERM * kStep + row / PERM);
  }
  __device__ __forceinline__ int64_t turn_at(int k, int row) const { return min(k, inner - 1) * ld + row; }
  __device__ __forceinline__ int64_t line_at(int u) const { return min(u / PIECES, rows - 1) * ld + u % PIECES * 8; }

  __device__ __forceinline__ void put(u32x4* lds) {
    // whether any load of this stage ended before its place
    const bool near = TR ? turn_at(8 * PIECES, ROWS) > total : (rows - 1) * ld + 8 * PIECES > total;
    const bool partial = inner < 8 * PIECES;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const bool in = kUnits % kThreads == 0 || q * kThreads + static_cast<int>(threadIdx.x) < kUnits;
      const int u = unit(q);
      if constexpr (TR) {
        const int row = u % (ROWS / 4) * 4, c = u / (ROWS / 4);
        if (near)
#pragma unroll
          for (int e = 0; e < 8; ++e) settle(r[q][e], turn_at(c * 8 + e, row), total);
        if constexpr (std::is_same_v<T, float>) {
          if (in)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
              F f;
#pragma unroll
              for (int e = 0; e < 8; ++e) f.v[e] = c * 8 + e < inner ? r[q][e].get(a) : 0.f;
              put_frag(lds, kPlane, place(row + a, c), f);
            }
        } else {
          if (partial)
#pragma unroll
            for (int e = 0; e < 8; ++e) cut(r[q][e], c * 8 + e < inner ? 4 : 0);
          if (in)
#pragma unroll
            for (int a = 0; a < 4; ++a) put_frag(lds, kPlane, place(row + a, c), column_of<F>(r[q], a));
        }
      } else {
        const int k = u % PIECES * 8;
        if (near) settle(r[q][0], line_at(u), total);
        if (partial) cut(r[q][0], inner - k);
        if (in) put_frag(lds, kPlane, place(u / PIECES, u % PIECES), frag_of<F>(r[q][0]));
      }
    }
  }

  static __device__ __forceinline__ F get(const u32x4* lds, int row, int c) {
    F f;
    get_frag(f, lds, kPlane, place(row, c));
    return f;
  }
};

// ---------------------------------------------------------------------------
// shrink: H[t, i] = sum_j W[i, j] x[t, j].  A workgroup takes a tile of 16 NT
// tokens and one of `parts` parts of the width, a stage of KB columns at a time.
// NT 4: a wave a token group and all ranks, or (ranks above 16) two token groups
// and half of the ranks, which reads the least from LDS.  NT 1 (short segments,
// where the weight is the traffic): the waves share the stage's columns and their
// sums meet in LDS in a fixed order.  W is [i][j] (AT false) or [j][i].
// Bound by the read of x and W, in practice by waits at the stages' barriers:
// bf16, rank 16, 8192 x 4096 19-20 us (3.8 TB/s); rank 64, 16384 x 8192 120 us
// (2.5 TB/s), 152 us with W as [j][i], turned in registers.
// ---------------------------------------------------------------------------
// Columns a stage: fewer where three terms of the weight take LDS and registers
// from a second and third workgroup of the compute unit (bf16 activations, float32
// weights: rank 64, 16384 x 8192, 64 columns 140 us, 128 180 us; rank 16, 6400 x
// 2048, 128 columns 12.7 us, 256 15.7 us; one token of 100, 256 columns 10.5 us,
// 512 12.9 us).
template <typename T, typename W, int RT, int NT>
constexpr int shrink_cols() {
  const bool three = kPlanes<Frag<T, W, true>> == 3;
  if (NT == 1) return three && RT < 4 ? 256 / RT : 512 / RT;
  if (three) return RT == 4 ? 64 : 128;
  return RT == 4 || kPlanes<Frag<T, T>> == 2 ? 128 : 256;
}

template <typename T, typename W, int RT, int NT, bool AT>
__global__ void __launch_bounds__(kThreads)
    shrink_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, int64_t ldw, Segs sg, int width,
                  int parts, int part, int rank, float* __restrict__ H, bool count_faults) {
  constexpr int KB = shrink_cols<T, W, RT, NT>(), PIECES = KB / 8;
  using SX = Stage<T, T, 16 * NT, PIECES, false, 1, true>;
  using SW = Stage<T, W, 16 * RT, PIECES, AT, AT ? 4 : 1, true>;
  __shared__ u32x4 lds[(SX::kBytes + SW::kBytes) / 16];
  u32x4* const ldw_ = lds + SX::kBytes / 16;
  const int tile = static_cast<int>(blockIdx.x) / parts, pt = static_cast<int>(blockIdx.x) % parts;
  const Tile tl = find_tile<16 * NT>(sg, tile, count_faults && pt == 0);
  if (tl.n <= 0) return;
  float* Hp = H + (static_cast<int64_t>(pt) * sg.tokens + tl.t0) * rank;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  if (tl.slot < 0) {
    for (int i = threadIdx.x; i < tl.n * rank; i += kThreads) Hp[i] = 0.f;
    return;
  }
  const int j0 = pt * part, j1 = min(width, j0 + part);
  const T* xs = x + static_cast<int64_t>(tl.t0) * ldx;
  const W* ws = w + tl.slot * ldw;
  const int64_t wld = AT ? rank : width;
  constexpr int RW = NT == 4 && RT >= 2 ? 2 : 1, UT = RW, UR = RT / RW;   // a wave's token groups and rank tiles
  const int tok = NT == 1 ? 0 : wave / RW * UT * 16, rk = NT == 1 ? 0 : wave % RW * UR;
  f32x4 acc[UT][UR] = {};
  SX sx;
  SW sw;
  const int64_t xall = (sg.tokens - 1 - tl.t0) * ldx + width, wall = static_cast<int64_t>(rank) * width;
  auto fetch = [&](int j) {
    const int64_t at = AT ? static_cast<int64_t>(j) * rank : j;
    sx.fetch(xs + j, ldx, tl.n, j1 - j, xall - j);
    sw.fetch(ws + at, wld, rank, j1 - j, wall - at);
  };
  if (j0 < j1) fetch(j0);
  for (int j = j0; j < j1; j += KB) {
    __syncthreads();
    sx.put(lds);
    sw.put(ldw_);
    __syncthreads();
    if (j + KB < j1) fetch(j + KB);
#pragma unroll
    for (int b = NT == 1 ? wave : 0; b < KB / 32; b += NT == 1 ? 4 : 1) {
      Frag<T, T> fx[UT];
#pragma unroll
      for (int u = 0; u < UT; ++u) fx[u] = SX::get(lds, tok + u * 16 + n, b * 4 + g);
#pragma unroll
      for (int r = 0; r < UR; ++r) {
        const auto fw = SW::get(ldw_, (rk + r) * 16 + n, b * 4 + g);
#pragma unroll
        for (int u = 0; u < UT; ++u) mma<true>(acc[u][r], fw, fx[u]);
      }
    }
  }
  if constexpr (NT == 1) {
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) sums[(wave * RT + r) * 64 + lane] = acc[0][r];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int r = 0; r < RT; ++r)
      for (int q = 1; q < 4; ++q) acc[0][r] += sums[(q * RT + r) * 64 + lane];
  }
#pragma unroll
  for (int u = 0; u < UT; ++u) {
    const int t = tok + u * 16 + n;
    if (t >= tl.n) continue;
#pragma unroll
    for (int r = 0; r < UR; ++r) {
      const int i = (rk + r) * 16 + g * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < rank) Hp[static_cast<int64_t>(t) * rank + i + e] = acc[u][r][e];
    }
  }
}

// ---------------------------------------------------------------------------
// expand: out[t, j] = base[t, j] + scale * sum_i W[i, j] H[t, i].  The products'
// rows are tokens and their columns n * PC + a of out, so a lane holds PC
// consecutive values of each of its 4 tokens and 16 lanes a stretch of a row.
// NT 4: a wave a token group, 128 columns of the weight staged for all of them
// (PC 8).  NT 1: a wave 64 of the 256 staged columns (PC 4).  W is [j][i] (AT true) or [i][j].
// Neighbouring workgroups take the column blocks of one tile: between them they
// read whole rows, not the same columns of many.  H comes in `parts` partial
// sums; the first column block also writes their sum to Hsum when that is asked.
// Bound by base and out: bf16, rank 16, 8192 x 4096 32-38 us (3.7-4.4 TB/s); rank
// 64, 16384 x 8192 151-155 us (3.7 TB/s).
// ---------------------------------------------------------------------------
template <int NT>
constexpr int kExpandCols = NT == 1 ? 256 : 128;

template <typename T, typename W, int RP, int NT, bool AT>
__global__ void __launch_bounds__(kThreads)
    expand_kernel(const T* base, int64_t ldb, const float* __restrict__ H, int parts, const W* __restrict__ w,
                  int64_t ldw, Segs sg, int width, int blocks, int span, int rank, float scale, T* out, int64_t ldo,
                  float* __restrict__ Hsum) {
  constexpr int COLS = kExpandCols<NT>, PC = NT == 1 ? 4 : 8, RK = (RP + 3) / 4;
  using SW = Stage<T, W, COLS, RP, !AT, PC, false>;                 // RP pieces of 8 ranks
  __shared__ u32x4 lds[SW::kBytes / 16];
  const int tile = static_cast<int>(blockIdx.x) / blocks, block = static_cast<int>(blockIdx.x) % blocks;
  const Tile tl = find_tile<16 * NT>(sg, tile, false);
  if (tl.n <= 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int c0 = block * span, c1 = min(width, c0 + span);
  const int64_t ball = (sg.tokens - 1) * ldb + width;    // elements of base
  if (tl.slot < 0) {
    if (Hsum != nullptr && block == 0)
      for (int i = threadIdx.x; i < tl.n * rank; i += kThreads) Hsum[static_cast<int64_t>(tl.t0) * rank + i] = 0.f;
    if (base == out) return;
    for (int t = wave; t < tl.n; t += 4)
      for (int j = c0 + lane * 8; j < c1; j += 512) {
        const int valid = min(8, c1 - j);
        Raw8<T> r = {};
        if (base != nullptr) {
          const int64_t at = (tl.t0 + t) * ldb + j;
          r = load_at<T, 8>(base, at, ball);
          settle(r, at, ball);
        }
        store_n(out + (tl.t0 + t) * ldo + j, r, valid);
      }
    return;
  }
  const W* ws = w + tl.slot * ldw;
  const int64_t wld = AT ? rank : width;
  const int64_t wall = static_cast<int64_t>(rank) * width;
  SW sw;
  auto fetch = [&](int j) {
    const int64_t at = AT ? static_cast<int64_t>(j) * rank : j;
    sw.fetch(ws + at, wld, width - j, rank, wall - at);
  };
  fetch(c0);
  const int tok = NT == 1 ? 0 : wave * 16;               // the wave's first token
  Frag<T, float> fh[RK];
#pragma unroll
  for (int b = 0; b < RK; ++b) {
    const int t = tok + n, i = b * 32 + g * 8;
    float h[8] = {};
    if (t < tl.n) {
      const int64_t at = static_cast<int64_t>(tl.t0 + t) * rank;
      for (int p = 0; p < parts; ++p) {
        // a load may take up to 7 floats behind the last part, which the workspace has
        const Raw8<float> q = load_n<float, 8>(H + p * sg.tokens * rank + at + min(i, rank - 1));
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] += i + e < rank ? q.get(e) : 0.f;
      }
      if (Hsum != nullptr && block == 0 && (NT == 4 || wave == 0))
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < rank) Hsum[at + i + e] = h[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) put2<float>(fh[b], e, f32x2{h[e] * scale, h[e + 1] * scale});
  }
  const int row = (NT == 1 ? wave * 64 : 0) + n * PC;    // this lane's columns of a stage
  auto base_at = [&](int q, int j0) { return (tl.t0 + min(tok + g * 4 + q, tl.n - 1)) * ldb + j0 + row; };
  RawN<T, PC> r[4] = {}, nxt[4] = {};
  if (base != nullptr)
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = load_at<T, PC>(base, base_at(q, c0), ball);
  for (int j0 = c0; j0 < c1; j0 += COLS) {
    const int j = j0 + row;
    __syncthreads();
    sw.put(lds);
    __syncthreads();
    if (j0 + COLS < c1) {
      fetch(j0 + COLS);
      if (base != nullptr)
#pragma unroll
        for (int q = 0; q < 4; ++q) nxt[q] = load_at<T, PC>(base, base_at(q, j0 + COLS), ball);
    }
    f32x4 acc[PC] = {};
#pragma unroll
    for (int b = 0; b < RK; ++b)
#pragma unroll
      for (int a = 0; a < PC; ++a) {
        // with fewer than 4 pieces the lanes of the others read the last one again: their h is 0,
        // and so are their weights
        Frag<T, W> fw = SW::get(lds, row + a, RP < 4 ? min(g, RP - 1) : b * 4 + g);
        if (RP < 4 && g >= RP) fw = Frag<T, W>{};
        mma<false>(acc[a], fh[b], fw);
      }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = tok + g * 4 + q;
      if (base != nullptr && j0 + COLS > c1) settle(r[q], base_at(q, j0), ball);
      if (t < tl.n) {
#pragma unroll
        for (int a = 0; a < PC; a += 2) {
          const f32x2 v = r[q].get2(a);
          r[q].set2(a, v[0] + acc[a][q], v[1] + acc[a + 1][q]);
        }
        store_n(out + (tl.t0 + t) * ldo + j, r[q], j0 + COLS <= c1 ? PC : c1 - j);
      }
      r[q] = nxt[q];
    }
  }
}

// ---------------------------------------------------------------------------
// outer: G_c[i, j] = scale * sum over the tokens t of slot c of H[t, i] x[t, j].
// The inner index is the token.  A workgroup takes one slot, every gridDim.z-th
// stage of 128 of its tokens, staged as H for its 4 waves, and 16 PC columns a
// wave: a lane loads PC columns of 8 tokens, the operands of PC products with
// columns n * PC + a.  With SPLIT the waves share 16 PC columns, take a quarter
// of each stage's tokens and add their sums in a fixed order: four times the
// workgroups where there are few.  With one part the sums go to G ([i][j], or
// [j][i] with AT), else each part's to its own copy (slot stride rank * width)
// for join_parts.  Bound by the read of x; 190-250 registers a lane leave two waves
// a SIMD: bf16, rank 64, 16384 x 8192 of 16 slots in 2 parts 141-152 us (2.4 TB/s);
// stages of 64 tokens 185 us.  A slot's segments are walked one after another, and
// the parts go by the average of tokens a slot: 16384 tokens of 4 clients in 4
// segments 31 us, in 512 152 us, in 8192 2.3 ms; 6400 tokens of 100 clients 88 us for
// the whole backward pass, 255 us where one of them has half.
// ---------------------------------------------------------------------------
constexpr int kOuterTokens = 128;
constexpr int kOuterCols = 4;

// the stages of a slot's tokens, segment by segment; every `turns`-th is this part's
struct SlotStages {
  const Segs& sg;
  int c, turn, turns;
  int s0 = -64, t = 0, t1 = 0;
  unsigned long long hits = 0;
  bool any = false;

  __device__ __forceinline__ bool next(int& at, int& left) {
    while (true) {
      for (; t < t1; t += kOuterTokens) {
        if (turn-- != 0) continue;
        turn = turns - 1;
        at = t;
        left = min(kOuterTokens, t1 - t);
        t += kOuterTokens;
        return true;
      }
      while (hits == 0) {
        s0 += 64;
        if (s0 >= sg.nseg) return false;
        const int s = s0 + static_cast<int>(threadIdx.x & 63);
        hits = __ballot(s < sg.nseg && sg.slots[min(s, sg.nseg - 1)] == c);
      }
      const int s = s0 + __ffsll(hits) - 1;
      hits &= hits - 1;
      t = seg_start(sg, s + 1);
      t1 = seg_start(sg, s + 2);
      any |= t1 > t;
    }
  }
};

template <typename T, int RT, bool AT, bool SPLIT>
__global__ void __launch_bounds__(kThreads)
    outer_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ H, Segs sg, int width, int rank,
                 float scale, float* __restrict__ G, int64_t ldg, int64_t part_stride, int accumulate) {
  using SH = Stage<T, float, 16 * RT, kOuterTokens / 8, true, 4, true>;
  constexpr int PC = kOuterCols, NB = SPLIT ? 1 : kOuterTokens / 32, kSums = SPLIT ? 2 * RT * PC * 64 : 0;
  __shared__ u32x4 lds[SH::kBytes / 16 > kSums ? SH::kBytes / 16 : kSums];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int c = blockIdx.y, block = static_cast<int>(blockIdx.x);
  const int j = ((SPLIT ? block : block * 4 + wave) * 16 + n) * PC, k0 = SPLIT ? wave * 32 : 0;
  const int valid = max(0, min(PC, width - j));
  const bool whole = (block + 1) * (SPLIT ? 16 : 64) * PC <= width;
  const int64_t xall = (sg.tokens - 1) * ldx + width;      // elements of x
  const int turns = static_cast<int>(gridDim.z);
  f32x4 acc[RT][PC] = {};
  SlotStages it{sg, c, static_cast<int>(blockIdx.z), turns};
  SH sh;
  RawN<T, PC> q[NB][8];
  int t, left;
  bool more = it.next(t, left);
  auto x_at = [&](int b, int e) { return static_cast<int64_t>(t + min(k0 + b * 32 + g * 8 + e, left - 1)) * ldx + j; };
  auto fetch = [&](int b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[b][e] = load_at<T, PC>(x, x_at(b, e), xall);
  };
  auto fetch_h = [&] {
    sh.fetch(H + static_cast<int64_t>(t) * rank, rank, rank, left, (sg.tokens - t) * rank);
  };
  if (more) {
    fetch_h();
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (k0 + b * 32 < left) fetch(b);
  }
  while (more) {
    __syncthreads();
    sh.put(lds);
    __syncthreads();
    const int t_now = t, left_now = left;
    more = it.next(t, left);
    if (more) fetch_h();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (k0 + b * 32 < left_now) {
        if (!whole)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            settle(q[b][e], static_cast<int64_t>(t_now + min(k0 + b * 32 + g * 8 + e, left_now - 1)) * ldx + j, xall);
        if (k0 + b * 32 + 32 > left_now)                     // no tokens of other segments
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k0 + b * 32 + g * 8 + e >= left_now) q[b][e] = RawN<T, PC>{};
        Frag<T, T> fx[PC];
#pragma unroll
        for (int a = 0; a < PC; ++a) fx[a] = column_of<Frag<T, T>>(q[b], a);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const auto fh = SH::get(lds, r * 16 + n, k0 / 8 + b * 4 + g);
#pragma unroll
          for (int a = 0; a < PC; ++a) mma<true>(acc[r][a], fh, fx[a]);
        }
      }
      if (more && k0 + b * 32 < left) fetch(b);                   // the next stage's into the registers just read
    }
  }
  if constexpr (SPLIT) {                                     // (0 + 2) + (1 + 3)
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half)
#pragma unroll
        for (int p = 0; p < RT * PC; ++p) sums[((wave - half) * RT * PC + p) * 64 + lane] = acc[p / PC][p % PC];
      __syncthreads();
      if (wave < half)
#pragma unroll
        for (int p = 0; p < RT * PC; ++p) acc[p / PC][p % PC] += sums[(wave * RT * PC + p) * 64 + lane];
    }
    if (wave != 0) return;
  }
  const bool any = it.any;
  const bool last = gridDim.z == 1;
  if (last && accumulate && !any) return;
  const bool add = last && accumulate;
  float* gc = G + blockIdx.z * part_stride + c * ldg;
  const float f = last ? scale : 1.f;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = r * 16 + g * 4 + q;
      if (i >= rank) continue;
#pragma unroll
      for (int a = 0; a < PC; ++a) {
        if (a >= valid) continue;
        float* p = gc + (AT ? static_cast<int64_t>(j + a) * rank + i : static_cast<int64_t>(i) * width + j + a);
        const float v = f * acc[r][a][q];
        *p = add ? *p + v : v;
      }
    }
}

// G_c = scale * sum of the parts, in order; 4 values a thread (two parts of 33.5
// MB: 21 us, 4.8 TB/s).  With accumulate every thread looks through the segments for
// one of its slot (512 segments: 60 us more; 8192: 0.85 ms more).
__global__ void __launch_bounds__(256)
    join_parts_kernel(const float* __restrict__ P, int parts, int64_t part_stride, Segs sg, int64_t per, float scale,
                      float* __restrict__ G, int64_t ldg, int accumulate) {
  const int c = blockIdx.y;
  const int64_t q = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (q >= per) return;
  if (accumulate) {
    bool any = false;
    for (int s = 0; s < sg.nseg; ++s) any |= sg.slots[s] == c && seg_start(sg, s + 2) > seg_start(sg, s + 1);
    if (!any) return;
  }
  const float* p = P + c * per;
  float a[4] = {};
  for (int z = 0; z < parts; ++z) {
    Raw4<float> r = load_at<float, 4>(p + z * part_stride, q, per);
    settle(r, q, per);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += r.get(e);
  }
  float* o = G + c * ldg + q;
  const int valid = static_cast<int>(min(per - q, int64_t{4}));
  Raw4<float> v;
#pragma unroll
  for (int e = 0; e < 4; e += 2)
    v.set2(e, (accumulate && e < valid ? o[e] : 0.f) + scale * a[e],
           (accumulate && e + 1 < valid ? o[e + 1] : 0.f) + scale * a[e + 1]);
  store_n(o, v, valid);
}

// ---------------------------------------------------------------------------
// The same three products element by element, for rows of fewer than 8 values
// (and outer for fewer than 8 hidden values), which the 16-byte loads above would
// read beyond.
// ---------------------------------------------------------------------------
template <typename T, typename W>
__global__ void __launch_bounds__(256)
    tiny_shrink_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, int64_t ldw, int64_t si,
                       int64_t sj, Segs sg, int width, int rank, float* __restrict__ H, bool count_faults) {
  const int64_t t = blockIdx.x;
  const int c = token_slot(sg.offsets, sg.slots, sg.nseg, sg.nslots, t, count_faults && threadIdx.x == 0);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = wave; i < rank; i += 4) {
    float a = 0.f;
    if (c >= 0) {
      for (int j = lane; j < width; j += 64) a += to_f32(w[c * ldw + i * si + j * sj]) * to_f32(x[t * ldx + j]);
      for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o);
    }
    if (lane == 0) H[t * rank + i] = a;
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
    tiny_expand_kernel(const T* base, int64_t ldb, const float* __restrict__ H, const W* __restrict__ w, int64_t ldw,
                       int64_t si, int64_t sj, Segs sg, int width, int rank, float scale, T* out, int64_t ldo) {
  const int64_t t = blockIdx.x;
  const int c = token_slot(sg.offsets, sg.slots, sg.nseg, sg.nslots, t, false);
  for (int j = threadIdx.x; j < width; j += 256) {
    const float b = base != nullptr ? to_f32(base[t * ldb + j]) : 0.f;
    float a = 0.f;
    if (c >= 0)
      for (int i = 0; i < rank; ++i) a += to_f32(w[c * ldw + i * si + j * sj]) * H[t * rank + i];
    out[t * ldo + j] = from_f32<T>(c >= 0 ? b + scale * a : b);
  }
}

__global__ void __launch_bounds__(256)
    tiny_sum_kernel(const float* H, int parts, int64_t all, float* sum) {
  const int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (q >= all) return;
  float a = H[q];
  for (int p = 1; p < parts; ++p) a += H[p * all + q];
  sum[q] = a;
}

template <typename T>
__global__ void __launch_bounds__(256)
    tiny_outer_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ H, Segs sg, int width, int rank,
                      float scale, float* __restrict__ G, int64_t ldg, int64_t si, int64_t sj, int accumulate) {
  const int c = blockIdx.y;
  const int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int j = static_cast<int>(q % width), i = static_cast<int>(q / width);
  if (i >= rank) return;
  float a = 0.f;
  bool any = false;
  for (int s = 0; s < sg.nseg; ++s) {
    if (sg.slots[s] != c) continue;
    const int t0 = seg_start(sg, s + 1), t1 = seg_start(sg, s + 2);
    for (int t = t0; t < t1; ++t) a += H[static_cast<int64_t>(t) * rank + i] * to_f32(x[t * ldx + j]);
    any |= t1 > t0;
  }
  float* g = G + c * ldg + i * si + j * sj;
  if (!accumulate) *g = scale * a;
  else if (any) *g += scale * a;
}

// the tokens of bad slots, for a gradient of B alone from given hidden values: no
// tile is searched for there
__global__ void __launch_bounds__(256) count_slots_kernel(Segs sg) {
  for (int i = threadIdx.x; i < sg.nseg; i += 256) {
    const int c = sg.slots[i], n = seg_start(sg, i + 2) - seg_start(sg, i + 1);
    if (n > 0 && (c < -1 || c >= sg.nslots)) count_row_fault(n);
  }
}

struct Shape {
  int64_t k, m;
  int rank;
  float scale;
};

static int check_common(const Segs& sg, const Shape& sh, const void* x, int64_t ldx, const void* A, int64_t lda,
                        const void* B, int64_t ldb, int32_t dtype, int32_t wdtype) {
  if (int rc = check_tokens(sg.tokens, sg.nslots)) return rc;
  if (int rc = check_segments(sg.offsets, sg.slots, sg.nseg)) return rc;
  if (int rc = check_dtype(dtype, "dtype")) return rc;
  SRA_REQUIRE(wdtype == SRA_F32 || wdtype == dtype, SRA_ERR_ARG,
              "wdtype must be SRA_F32 or the activations' dtype, got %d", wdtype);
  SRA_REQUIRE((x != nullptr || sg.tokens == 0) && A != nullptr && B != nullptr, SRA_ERR_ARG, "x, A and B must be non-null");
  SRA_REQUIRE(sh.k >= 1 && sh.m >= 1 && sh.k < (int64_t{1} << 28) && sh.m < (int64_t{1} << 28), SRA_ERR_SHAPE,
              "k and m must be in [1, 2^28), got %lld, %lld", static_cast<long long>(sh.k),
              static_cast<long long>(sh.m));
  SRA_REQUIRE(sh.rank >= 1, SRA_ERR_ARG, "rank must be >= 1, got %d", sh.rank);
  SRA_REQUIRE(sh.rank <= SRA_ADAPTER_MAX_RANK, SRA_ERR_UNSUPPORTED, "rank %d is above %d", sh.rank,
              SRA_ADAPTER_MAX_RANK);
  SRA_REQUIRE(ldx >= sh.k || sg.tokens <= 1, SRA_ERR_SHAPE, "x needs a row stride >= %lld, got %lld",
              static_cast<long long>(sh.k), static_cast<long long>(ldx));
  SRA_REQUIRE(sg.nslots == 1 || (lda >= sh.rank * sh.k && ldb >= sh.rank * sh.m), SRA_ERR_SHAPE,
              "A and B need slot strides >= rank * k and rank * m");
  return SRA_OK;
}

// ---------------------------------------------------------------------------
// Plans
// ---------------------------------------------------------------------------
constexpr int kMaxParts = 16;

// Token groups of 16 a tile: 4 where segments are long enough to fill half of
// them on average, else 1 (100 segments, 2048 wide, rank 16, bf16: 16 tokens a
// segment 21.3 us with 1, 24.0 with 4; 32 tokens 27.3, 27.6; 64 tokens 41.9, 36.9).
static int tile_groups(int64_t tokens, int nseg) { return tokens >= 32 * static_cast<int64_t>(nseg) ? 4 : 1; }

// Parts of the width that shrink sums apart: two workgroups a compute unit where
// the tiles alone give fewer, a part never below 512 columns.  Where even one a
// unit is out of reach, tiles of 64 tokens go down to 256 columns, or 128 at ranks
// whose partial sums expand reads cheaply (a float32 step of 1501 tokens, 1001 ->
// 777, rank 5: 70 us with 512, 60 with 256, 56 with 128; 2203 tokens, 960 -> 1216,
// rank 19: 96, 85, 85; 2048 bf16 tokens, 1024 wide, rank 64: 23.5, 23.1, 25.9).
static int shrink_parts(int64_t tokens, int nseg, int64_t width, int rank) {
  const int groups = tile_groups(tokens, nseg);
  const int64_t tiles = tokens / (16 * groups) + std::min<int64_t>(nseg, tokens);
  const int64_t few = groups == 4 ? (rank <= 16 ? 256 : 512) : 1024;
  int p = 1;
  while (p < kMaxParts && ((tiles * p < 256 && width >= few * p) || (tiles * p < 512 && width >= 1024 * p))) p *= 2;
  return p;
}

// Whether outer's waves share their columns: where whole workgroups' columns give
// fewer than one workgroup a compute unit (1501 tokens of 13 slots, 1001 wide: 11.5
// us, 22.5 us without; with 800 workgroups 28 us, 24 us without).
static bool outer_split(int nslots, int64_t width) { return cdiv(width, 64 * kOuterCols) * nslots < 256; }

// Parts of a client's tokens that outer sums apart: four workgroups a compute
// unit, each with at least 2 stages of tokens on average (clients with more hold
// the launch up less, the join costs a pass over the parts).
static int outer_parts(int64_t tokens, int nslots, int64_t width) {
  const int64_t blocks = cdiv(width, (outer_split(nslots, width) ? 16 : 64) * kOuterCols) * nslots;
  const int64_t stages = cdiv(tokens, kOuterTokens * static_cast<int64_t>(nslots));
  int p = 1;
  while (p < kMaxParts && blocks * p < 1024 && stages >= 2 * p) p *= 2;
  return p;
}

struct Workspace {
  size_t h, z, ga, gb, bytes;
};

static Workspace plan(int64_t tokens, int nseg, int nslots, int64_t k, int64_t m, int rank) {
  const size_t row = static_cast<size_t>(rank) * 4;
  const int pa = outer_parts(tokens, nslots, k), pb = outer_parts(tokens, nslots, m);
  Workspace w{};
  w.h = 0;
  // expand may load up to 7 floats behind the parts of h or z
  w.z = w.h + static_cast<size_t>(tokens) * row * shrink_parts(tokens, nseg, k, rank) + 32;
  w.ga = w.z + static_cast<size_t>(tokens) * row * (shrink_parts(tokens, nseg, m, rank) + 1) + 32;
  w.gb = w.ga + (pa > 1 ? static_cast<size_t>(pa) * nslots * k * row : 0);
  w.bytes = w.gb + (pb > 1 ? static_cast<size_t>(pb) * nslots * m * row : 0) + 16;
  return w;
}

// f(groups, rank tiles) as constants
template <typename F>
static int with_tile(const Segs& sg, int rank, F&& f) {
  auto ranks = [&](auto nt) {
    if (rank <= 16) return f(nt, std::integral_constant<int, 1>{});
    if (rank <= 32) return f(nt, std::integral_constant<int, 2>{});
    return f(nt, std::integral_constant<int, 4>{});
  };
  return tile_groups(sg.tokens, sg.nseg) == 4 ? ranks(std::integral_constant<int, 4>{})
                                              : ranks(std::integral_constant<int, 1>{});
}

template <typename T, typename W, bool AT>
static int launch_shrink(const void* x, int64_t ldx, const void* w, int64_t ldw, const Segs& sg, int64_t width,
                         int parts, int rank, float* H, bool count_faults, hipStream_t st) {
  if (width < 8) {
    if (int rc = check_launch(sg.tokens, 256)) return rc;
    hipLaunchKernelGGL((tiny_shrink_kernel<T, W>), dim3(static_cast<unsigned>(sg.tokens)), dim3(256), 0, st,
                       static_cast<const T*>(x), ldx, static_cast<const W*>(w), ldw, AT ? 1 : width,
                       AT ? static_cast<int64_t>(rank) : 1, sg, static_cast<int>(width), rank, H, count_faults);
    return launch_status("tiny_shrink_kernel");
  }
  return with_tile(sg, rank, [&](auto nt, auto rt) {
    constexpr int NT = decltype(nt)::value, RT = decltype(rt)::value, KB = shrink_cols<T, W, RT, NT>();
    const int part = static_cast<int>(cdiv(cdiv(width, parts), KB) * KB);
    if (int rc = check_launch(static_cast<int64_t>(tile_count<16 * NT>(sg)) * parts, kThreads)) return rc;
    hipLaunchKernelGGL((shrink_kernel<T, W, RT, NT, AT>), dim3(tile_count<16 * NT>(sg) * parts), dim3(kThreads), 0, st,
                       static_cast<const T*>(x), ldx, static_cast<const W*>(w), ldw, sg, static_cast<int>(width),
                       parts, part, rank, H, count_faults);
    return launch_status("shrink_kernel");
  });
}

template <typename T, typename W, bool AT>
static int launch_expand(const void* base, int64_t ldb, const float* H, int parts, const void* w, int64_t ldw,
                         const Segs& sg, int64_t width, int rank, float scale, void* out, int64_t ldo, float* Hsum,
                         hipStream_t st) {
  if (width < 8) {
    if (int rc = check_launch(sg.tokens, 256)) return rc;
    if (parts > 1 || Hsum != nullptr) {
      float* sum = Hsum != nullptr ? Hsum : const_cast<float*>(H);
      const int64_t all = sg.tokens * rank;
      hipLaunchKernelGGL(tiny_sum_kernel, dim3(static_cast<unsigned>(cdiv(all, 256))), dim3(256), 0, st, H, parts, all,
                         sum);
      if (int rc = launch_status("tiny_sum_kernel")) return rc;
      H = sum;
    }
    hipLaunchKernelGGL((tiny_expand_kernel<T, W>), dim3(static_cast<unsigned>(sg.tokens)), dim3(256), 0, st,
                       static_cast<const T*>(base), ldb, H, static_cast<const W*>(w), ldw, AT ? 1 : width,
                       AT ? static_cast<int64_t>(rank) : 1, sg, static_cast<int>(width), rank, scale,
                       static_cast<T*>(out), ldo);
    return launch_status("tiny_expand_kernel");
  }
  return with_tile(sg, rank, [&](auto nt, auto rt) {
    constexpr int NT = decltype(nt)::value, RT = decltype(rt)::value, COLS = kExpandCols<NT>;
    const int tiles = tile_count<16 * NT>(sg);
    // Four workgroups a compute unit where the width allows it; with tiles of 64
    // tokens up to 16 if each keeps two stages, so that uneven tiles leave less
    // behind (16384 tokens of 16 clients, 8192 wide, rank 64: 170 us, 178 us with
    // four; 6400 tokens of 100, 2048 wide, rank 16: 28.5 us, 31 us with four, 37 us
    // with single stages).
    int64_t want = std::min<int64_t>(cdiv(1024, tiles), cdiv(width, COLS));
    if (NT == 4) want = std::max(want, std::min<int64_t>(cdiv(4096, tiles), cdiv(width, 2 * COLS)));
    const int span = static_cast<int>(cdiv(cdiv(width, want), COLS) * COLS);
    const int blocks = static_cast<int>(cdiv(width, span));
    if (int rc = check_launch(static_cast<int64_t>(tiles) * blocks, kThreads)) return rc;
    auto go = [&](auto rp) {
      constexpr int RP = decltype(rp)::value;
      hipLaunchKernelGGL((expand_kernel<T, W, RP, NT, AT>), dim3(static_cast<unsigned>(tiles) * blocks),
                         dim3(kThreads), 0, st, static_cast<const T*>(base), ldb, H, parts, static_cast<const W*>(w),
                         ldw, sg, static_cast<int>(width), blocks, span, rank, scale, static_cast<T*>(out), ldo, Hsum);
      return launch_status("expand_kernel");
    };
    if constexpr (RT == 1) return rank <= 8 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
    else return go(std::integral_constant<int, 2 * RT>{});
  });
}

// whether a gradient of so many tokens is summed element by element
static bool outer_tiny(int64_t tokens, int64_t width, int rank) { return width < 8 || tokens * rank < 8; }

// the largest of launch_outer's grids, which go by the weight's size alone where
// there are no tokens
static int check_outer(const Segs& sg, int64_t width, int rank) {
  const int64_t per = rank * width;
  return check_launch(outer_tiny(sg.tokens, width, rank) ? cdiv(per, 256) : cdiv(per, 1024), 256);
}

template <typename T, bool AT>
static int launch_outer(const void* x, int64_t ldx, const float* H, const Segs& sg, int64_t width, int rank,
                        float scale, float* G, int64_t ldg, int accumulate, float* parts_ws, hipStream_t st) {
  if (outer_tiny(sg.tokens, width, rank)) {
    const dim3 tg(static_cast<unsigned>(cdiv(rank * width, 256)), static_cast<unsigned>(sg.nslots));
    hipLaunchKernelGGL((tiny_outer_kernel<T>), tg, dim3(256), 0, st, static_cast<const T*>(x), ldx, H, sg,
                       static_cast<int>(width), rank, scale, G, ldg, AT ? 1 : width,
                       AT ? static_cast<int64_t>(rank) : 1, accumulate);
    return launch_status("tiny_outer_kernel");
  }
  const int parts = outer_parts(sg.tokens, sg.nslots, width);
  const int64_t per = rank * width, stride = per * sg.nslots;
  const int rc = with_tile(sg, rank, [&](auto, auto rt) {
    constexpr int RT = decltype(rt)::value;
    auto go = [&](auto split) {
      constexpr bool SPLIT = decltype(split)::value;
      const dim3 grid(static_cast<unsigned>(cdiv(width, (SPLIT ? 16 : 64) * kOuterCols)),
                      static_cast<unsigned>(sg.nslots), parts);
      hipLaunchKernelGGL((outer_kernel<T, RT, AT, SPLIT>), grid, dim3(kThreads), 0, st, static_cast<const T*>(x), ldx,
                         H, sg, static_cast<int>(width), rank, scale, parts > 1 ? parts_ws : G, parts > 1 ? per : ldg,
                         stride, accumulate);
      return launch_status("outer_kernel");
    };
    return outer_split(sg.nslots, width) ? go(std::true_type{}) : go(std::false_type{});
  });
  if (rc || parts == 1) return rc;
  const dim3 jg(static_cast<unsigned>(cdiv(per, 1024)), static_cast<unsigned>(sg.nslots));
  hipLaunchKernelGGL(join_parts_kernel, jg, dim3(256), 0, st, parts_ws, parts, stride, sg, per, scale, G, ldg,
                     accumulate);
  return launch_status("join_parts_kernel");
}

struct Weights {
  const void* A;
  int64_t lda;
  const void* B;
  int64_t ldb;
};

template <typename T, typename W>
static int run_apply(const void* base, int64_t ldbase, const void* x, int64_t ldx, const Weights& w, const Segs& sg,
                     const Shape& sh, void* out, int64_t ldo, float* hidden, char* ws, hipStream_t st) {
  const int parts = shrink_parts(sg.tokens, sg.nseg, sh.k, sh.rank);
  float* H = reinterpret_cast<float*>(ws);
  if (int rc = launch_shrink<T, W, false>(x, ldx, w.A, w.lda, sg, sh.k, parts, sh.rank, H, true, st)) return rc;
  return launch_expand<T, W, true>(base, ldbase, H, parts, w.B, w.ldb, sg, sh.m, sh.rank, sh.scale, out, ldo,
                                   hidden, st);
}

struct GradOut {
  const float* hidden;
  const void* dxbase;
  int64_t lddxb;
  void* dx;
  int64_t lddx;
  float* dA;
  int64_t ldda;
  float* dB;
  int64_t lddb;
  int accumulate;
};

template <typename T, typename W>
static int run_grad(const void* dout, int64_t lddo, const void* x, int64_t ldx, const Weights& w, const Segs& sg,
                    const Shape& sh, const GradOut& g, char* ws, const Workspace& pl, hipStream_t st) {
  const float* H = g.hidden;
  float* Hw = reinterpret_cast<float*>(ws + pl.h);
  float* Z = reinterpret_cast<float*>(ws + pl.z);
  if (sg.tokens > 0) {
    if (g.dx != nullptr || g.dA != nullptr) {
      // the parts of z meet in the expand that needs them; without one there is one part
      const int parts = g.dx != nullptr ? shrink_parts(sg.tokens, sg.nseg, sh.m, sh.rank) : 1;
      float* Zp = Z;
      if (parts > 1) Z = Zp + static_cast<int64_t>(parts) * sg.tokens * sh.rank;
      if (int rc = launch_shrink<T, W, true>(dout, lddo, w.B, w.ldb, sg, sh.m, parts, sh.rank, Zp, true, st)) return rc;
      if (g.dx != nullptr)
        if (int rc = launch_expand<T, W, false>(g.dxbase, g.lddxb, Zp, parts, w.A, w.lda, sg, sh.k, sh.rank, sh.scale,
                                                g.dx, g.lddx, parts > 1 ? Z : nullptr, st))
          return rc;
    }
    const bool counted = g.dx != nullptr || g.dA != nullptr;
    if (g.dB != nullptr && H == nullptr) {
      H = Hw;
      if (int rc = launch_shrink<T, W, false>(x, ldx, w.A, w.lda, sg, sh.k, 1, sh.rank, Hw, !counted, st)) return rc;
    } else if (!counted) {
      hipLaunchKernelGGL(count_slots_kernel, dim3(1), dim3(256), 0, st, sg);
      if (int rc = launch_status("count_slots_kernel")) return rc;
    }
  }
  if (g.dA != nullptr)
    if (int rc = launch_outer<T, false>(x, ldx, Z, sg, sh.k, sh.rank, sh.scale, g.dA, g.ldda, g.accumulate,
                                        reinterpret_cast<float*>(ws + pl.ga), st))
      return rc;
  if (g.dB != nullptr)
    return launch_outer<T, true>(dout, lddo, H, sg, sh.m, sh.rank, sh.scale, g.dB, g.lddb, g.accumulate,
                                 reinterpret_cast<float*>(ws + pl.gb), st);
  return SRA_OK;
}

// f(T{}, W{}) for the activations' and the weights' types
template <typename F>
static int with_types(int32_t dtype, int32_t wdtype, F&& f) {
  if (dtype == SRA_F32) return f(float{}, float{});
  if (dtype == SRA_BF16) return wdtype == SRA_F32 ? f(__bf16{}, float{}) : f(__bf16{}, __bf16{});
  return wdtype == SRA_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
}

}  // namespace sra

using namespace sra;

extern "C" int sra_adapter_workspace_bytes(int64_t tokens, int32_t nseg, int32_t nslots, int64_t k, int64_t m,
                                           int32_t rank, size_t* bytes) {
  SRA_REQUIRE(bytes != nullptr, SRA_ERR_ARG, "null bytes pointer");
  if (int rc = check_tokens(tokens, nslots)) return rc;
  SRA_REQUIRE(nseg >= 0, SRA_ERR_ARG, "nseg must be >= 0, got %d", nseg);
  SRA_REQUIRE(k >= 1 && m >= 1 && k < (int64_t{1} << 28) && m < (int64_t{1} << 28), SRA_ERR_SHAPE,
              "k and m must be in [1, 2^28), got %lld, %lld", static_cast<long long>(k), static_cast<long long>(m));
  SRA_REQUIRE(rank >= 1, SRA_ERR_ARG, "rank must be >= 1, got %d", rank);
  SRA_REQUIRE(rank <= SRA_ADAPTER_MAX_RANK, SRA_ERR_UNSUPPORTED, "rank %d is above %d", rank,
              SRA_ADAPTER_MAX_RANK);
  *bytes = plan(tokens, nseg, nslots, k, m, rank).bytes;
  return SRA_OK;
}

extern "C" int sra_adapter_apply(const void* base, int64_t ldbase, const void* x, int64_t ldx, const void* A,
                                 int64_t lda, const void* B, int64_t ldb, const int64_t* offsets,
                                 const int32_t* slots, int32_t nseg, int64_t tokens, int32_t nslots, int64_t k,
                                 int64_t m, int32_t rank, float scale, int32_t dtype, int32_t wdtype, void* out,
                                 int64_t ldo, float* hidden, void* ws, size_t ws_bytes, void* stream) {
  const Segs sg{offsets, slots, nseg, nslots, tokens};
  const Shape sh{k, m, rank, scale};
  if (int rc = check_common(sg, sh, x, ldx, A, lda, B, ldb, dtype, wdtype)) return rc;
  SRA_REQUIRE(out != nullptr || tokens == 0, SRA_ERR_ARG, "out must be non-null");
  SRA_REQUIRE(tokens <= 1 || (ldo >= m && (base == nullptr || ldbase >= m)), SRA_ERR_SHAPE,
              "base and out need row strides >= m");
  SRA_REQUIRE(base != out || ldbase == ldo || tokens <= 1, SRA_ERR_SHAPE, "base and out are one buffer with two row strides");
  if (tokens == 0) return SRA_OK;
  size_t need = 0;
  if (int rc = sra_adapter_workspace_bytes(tokens, nseg, nslots, k, m, rank, &need)) return rc;
  SRA_REQUIRE(ws != nullptr && ws_bytes >= need, SRA_ERR_WORKSPACE, "adapter workspace: need %zu bytes, got %zu", need,
              ws_bytes);
  const Weights wt{A, lda, B, ldb};
  return with_types(dtype, wdtype, [&](auto t, auto w) {
    return run_apply<decltype(t), decltype(w)>(base, ldbase, x, ldx, wt, sg, sh, out, ldo, hidden,
                                               static_cast<char*>(ws), static_cast<hipStream_t>(stream));
  });
}

extern "C" int sra_adapter_grad(const void* dout, int64_t lddo, const void* x, int64_t ldx, const void* A,
                                int64_t lda, const void* B, int64_t ldb, const int64_t* offsets,
                                const int32_t* slots, int32_t nseg, int64_t tokens, int32_t nslots, int64_t k,
                                int64_t m, int32_t rank, float scale, int32_t dtype, int32_t wdtype,
                                const float* hidden, const void* dxbase, int64_t lddxb, void* dx, int64_t lddx,
                                float* dA, int64_t ldda, float* dB, int64_t lddb, int32_t accumulate, void* ws,
                                size_t ws_bytes, void* stream) {
  const Segs sg{offsets, slots, nseg, nslots, tokens};
  const Shape sh{k, m, rank, scale};
  if (int rc = check_common(sg, sh, x, ldx, A, lda, B, ldb, dtype, wdtype)) return rc;
  SRA_REQUIRE(dout != nullptr || tokens == 0, SRA_ERR_ARG, "dout must be non-null");
  SRA_REQUIRE(tokens <= 1 || lddo >= m, SRA_ERR_SHAPE, "dout needs a row stride >= m");
  SRA_REQUIRE(dx == nullptr || tokens <= 1 || (lddx >= k && (dxbase == nullptr || lddxb >= k)), SRA_ERR_SHAPE,
              "dxbase and dx need row strides >= k");
  SRA_REQUIRE(dx == nullptr || dxbase != dx || lddxb == lddx || tokens <= 1, SRA_ERR_SHAPE,
              "dxbase and dx are one buffer with two row strides");
  SRA_REQUIRE(nslots == 1 || ((dA == nullptr || ldda >= rank * k) && (dB == nullptr || lddb >= rank * m)),
              SRA_ERR_SHAPE, "dA and dB need slot strides >= rank * k and rank * m");
  SRA_REQUIRE((dA == nullptr && dB == nullptr) || nslots <= 65535, SRA_ERR_UNSUPPORTED,
              "gradients of %d slots: more than 65535", nslots);
  if (dx == nullptr && dA == nullptr && dB == nullptr) return SRA_OK;
  size_t need = 0;
  if (int rc = sra_adapter_workspace_bytes(tokens, nseg, nslots, k, m, rank, &need)) return rc;
  SRA_REQUIRE(ws != nullptr && ws_bytes >= need, SRA_ERR_WORKSPACE, "adapter workspace: need %zu bytes, got %zu", need,
              ws_bytes);
  SRA_REQUIRE(dx == nullptr || (dx != dout && dx != x), SRA_ERR_ARG, "dx must not be dout or x: they are read after it");
  if (dA != nullptr)
    if (int rc = check_outer(sg, k, rank)) return rc;
  if (dB != nullptr)
    if (int rc = check_outer(sg, m, rank)) return rc;
  const GradOut g{hidden, dxbase, lddxb, dx, lddx, dA, ldda, dB, lddb, accumulate};
  const Weights wt{A, lda, B, ldb};
  return with_types(dtype, wdtype, [&](auto t, auto w) {
    return run_grad<decltype(t), decltype(w)>(dout, lddo, x, ldx, wt, sg, sh, g, static_cast<char*>(ws),
                                              plan(tokens, nseg, nslots, k, m, rank), static_cast<hipStream_t>(stream));
  });
}

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
// (v_mfma_f32_16x16x32_bf16): bf16 values as they are, float32 and fp16 ones
// (weights, h, z, fp16 activations) as two bf16 terms, the nearest and the rest,
// with the product of the two rests left out: 2^-16 of a product, far inside
// the rounding of 16-bit activations, for at most three matrix instructions
// where memory leaves room for more.  A product with an infinity is then the sum
// of two that may have opposite signs: it comes out infinite or NaN.  float32 activations run on the float32
// units (v_mfma_f32_16x16x4_f32).
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
template <typename S>
struct Raw8 {
  S v[8];
};

// 8 consecutive elements at any alignment of their type (the hardware's global
// loads take it); valid < 8 leaves the rest zero
template <typename S>
__device__ __forceinline__ Raw8<S> load8(const S* p) {
  typedef u32x4 __attribute__((aligned(2))) any_u32x4;
  Raw8<S> r;
  const any_u32x4* q = reinterpret_cast<const any_u32x4*>(p);
  u32x4* o = reinterpret_cast<u32x4*>(&r);
  o[0] = q[0];
  if constexpr (sizeof(S) == 4) o[1] = q[1];
  return r;
}

template <typename S>
__device__ __forceinline__ Raw8<S> load8(const S* p, int64_t valid) {
  if (valid >= 8) return load8(p);
  Raw8<S> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = e < valid ? p[e] : static_cast<S>(0.f);
  return r;
}

template <typename S>
__device__ __forceinline__ Raw8<S> load8_strided(const S* p, int64_t stride, int64_t valid) {
  Raw8<S> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = e < valid ? p[e * stride] : static_cast<S>(0.f);
  return r;
}

template <typename S>
__device__ __forceinline__ void store8(S* p, const Raw8<S>& r, int64_t valid) {
  typedef u32x4 __attribute__((aligned(2))) any_u32x4;
  if (valid >= 8) {
    any_u32x4* q = reinterpret_cast<any_u32x4*>(p);
    const u32x4* o = reinterpret_cast<const u32x4*>(&r);
    q[0] = o[0];
    if constexpr (sizeof(S) == 4) q[1] = o[1];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) p[e] = r.v[e];
  }
}

template <int N>
struct Terms {
  bf16x8 t[N];
};

// nearest bf16 and the rest
__device__ __forceinline__ void split_into(Terms<2>& f, int e, float x) {
  const __bf16 hi = static_cast<__bf16>(x);
  const float h = static_cast<float>(hi);
  f.t[0][e] = hi;
  f.t[1][e] = static_cast<__bf16>(x - h);
}

// the operand that T's matrix units take for stored values S
template <typename T, typename S>
using Frag = std::conditional_t<std::is_same_v<T, float>, Raw8<float>,
                                Terms<std::is_same_v<S, __bf16> ? 1 : 2>>;

template <typename T, typename S>
__device__ __forceinline__ void put_elem(Frag<T, S>& f, int e, S x) {
  if constexpr (std::is_same_v<T, float>) f.v[e] = x;
  else if constexpr (std::is_same_v<S, __bf16>) f.t[0][e] = x;
  else split_into(f, e, static_cast<float>(x));
}

template <typename T, typename S>
__device__ __forceinline__ Frag<T, S> frag_of(const Raw8<S>& r) {
  Frag<T, S> f;
#pragma unroll
  for (int e = 0; e < 8; ++e) put_elem<T, S>(f, e, r.v[e]);
  return f;
}

template <int N, int M>
__device__ __forceinline__ void mma(f32x4& acc, const Terms<N>& a, const Terms<M>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
#pragma unroll
    for (int j = M - 1; j >= 0; --j)
      if (i + j < 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[i], b.t[j], acc, 0, 0, 0);
}

__device__ __forceinline__ void mma(f32x4& acc, const Raw8<float>& a, const Raw8<float>& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Token tiles.  Segments are cut into tiles of TT tokens that never cross a
// segment.  Segment i starts at e_i, so its tiles may take the numbers from
// e_i / TT + i on: e_{i+1} / TT + i + 1 is never below the last of them.  A
// workgroup finds its tile on the device by searching those numbers; the rows
// before the first and behind the last segment count as segments without a slot.
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
__device__ __forceinline__ Tile find_tile(const Segs& sg, int tile) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = sg.nseg + 2;
  while (len > 1) {                          // 64 candidates at a time
    const int step = (len + 63) >> 6, i = lane * step;
    const bool at = i < len && seg_start(sg, lo + i) / TT + lo + i <= tile;
    const int hits = max(__popcll(__ballot(at)), 1);
    const int skip = (hits - 1) * step;
    lo += skip;
    len = min(step, len - skip);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int first = seg_start(sg, lo);
  // numbers that no tile has end here, and so do offsets that do not ascend
  const int64_t t0 = first + static_cast<int64_t>(tile - first / TT - lo) * TT;
  const int64_t left = seg_start(sg, lo + 1) - t0;
  Tile t;
  t.t0 = static_cast<int>(t0);
  t.n = t0 < first ? 0 : static_cast<int>(max(int64_t{0}, min(left, int64_t{TT})));
  t.slot = lo == 0 || lo == sg.nseg + 1 || t.n <= 0 ? -1 : checked_slot(sg.slots, lo - 1, sg.nslots);
  return t;
}

template <int TT>
static int tile_count(const Segs& sg) {
  return static_cast<int>(sg.tokens / TT) + sg.nseg + 2;
}

// ---------------------------------------------------------------------------
// shrink: H[t, i] = sum_j W[i, j] x[t, j].  A workgroup of 16 waves takes a tile
// of 16 NT tokens and one of gridDim.y parts of the width; a wave takes one rank
// tile and every (16 / rank tiles)-th stretch of 32, and the waves' sums meet in
// LDS.  W is stored [i][j] (AT false) or [j][i] (AT true).
// ---------------------------------------------------------------------------
constexpr int kShrinkWaves = 16;

template <typename T, typename W, int NT, bool AT>
__global__ void __launch_bounds__(kShrinkWaves * 64)
    shrink_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, int64_t ldw, Segs sg, int width,
                  int part, int rank, float* __restrict__ H) {
  __shared__ f32x4 sums[kShrinkWaves][NT][64];
  const Tile tl = find_tile<16 * NT>(sg, blockIdx.x);
  if (tl.n <= 0) return;
  float* Hp = H + (static_cast<int64_t>(blockIdx.y) * sg.tokens + tl.t0) * rank;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  if (tl.slot < 0) {
    for (int i = threadIdx.x; i < tl.n * rank; i += kShrinkWaves * 64) Hp[i] = 0.f;
    return;
  }
  const int rtiles = (rank + 15) >> 4, parts = kShrinkWaves / rtiles;
  const int rt = wave % rtiles, kp = wave / rtiles;
  f32x4 acc[NT] = {};
  if (kp < parts) {
    const int j0 = static_cast<int>(blockIdx.y) * part, j1 = min(width, j0 + part);
    const int i = min(rt * 16 + n, rank - 1);            // rows beyond the rank are not stored
    const W* wp = w + tl.slot * ldw + (AT ? static_cast<int64_t>(i) : static_cast<int64_t>(i) * width);
    const T* xp[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) xp[u] = x + (tl.t0 + min(u * 16 + n, tl.n - 1)) * ldx;
    const int full = (j1 - j0) / 32;
#pragma unroll 4
    for (int b = kp; b < full; b += parts) {
      const int j = j0 + b * 32 + g * 8;
      const Frag<T, W> fw = AT ? frag_of<T, W>(load8_strided(wp + static_cast<int64_t>(j) * rank, rank, 8))
                               : frag_of<T, W>(load8(wp + j));
#pragma unroll
      for (int u = 0; u < NT; ++u) mma(acc[u], fw, frag_of<T, T>(load8(xp[u] + j)));
    }
    if (j0 + full * 32 < j1 && kp == full % parts) {
      const int j = j0 + full * 32 + g * 8, valid = max(0, min(8, j1 - j));
      const Frag<T, W> fw = AT ? frag_of<T, W>(load8_strided(wp + static_cast<int64_t>(j) * rank, rank, valid))
                               : frag_of<T, W>(load8(wp + j, valid));
#pragma unroll
      for (int u = 0; u < NT; ++u) mma(acc[u], fw, frag_of<T, T>(load8(xp[u] + j, valid)));
    }
  }
#pragma unroll
  for (int u = 0; u < NT; ++u) sums[wave][u][lane] = acc[u];
  __syncthreads();
  for (int q = wave; q < rtiles * NT; q += kShrinkWaves) {
    const int r = q % rtiles, u = q / rtiles;
    f32x4 a = sums[r][u][lane];
    for (int p = 1; p < parts; ++p) a += sums[p * rtiles + r][u][lane];
    const int t = u * 16 + n, i = r * 16 + g * 4;
    if (t < tl.n) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < rank) Hp[static_cast<int64_t>(t) * rank + i + e] = a[e];
    }
  }
}

// ---------------------------------------------------------------------------
// expand: out[t, j] = base[t, j] + scale * sum_i W[i, j] H[t, i].  A wave takes
// a tile of 16 NT tokens and, step by step, 128 columns.  W is stored [j][i]
// (AT true) or [i][j] (AT false).  The product's rows are columns of out,
// permuted so that a lane holds runs of 8 consecutive ones of its token.
// H comes in `parts` partial sums; the first column block also writes their sum
// to Hsum when that is asked.
// ---------------------------------------------------------------------------
constexpr int kExpandCols = 128;

template <typename T, typename W, int RK, int NT, bool AT>
__global__ void __launch_bounds__(256)
    expand_kernel(const T* base, int64_t ldb, const float* __restrict__ H, int parts, const W* __restrict__ w,
                  int64_t ldw, Segs sg, int width, int span, int rank, float scale, T* out, int64_t ldo,
                  float* __restrict__ Hsum) {
  const Tile tl = find_tile<16 * NT>(sg, blockIdx.x);
  if (tl.n <= 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int c0 = static_cast<int>(blockIdx.y) * span, c1 = min(width, c0 + span);
  if (tl.slot < 0) {
    if (Hsum != nullptr && blockIdx.y == 0)
      for (int i = threadIdx.x; i < tl.n * rank; i += 256) Hsum[static_cast<int64_t>(tl.t0) * rank + i] = 0.f;
    if (base == out) return;
    for (int t = wave; t < tl.n; t += 4)
      for (int j = c0 + lane * 8; j < c1; j += 512) {
        const int valid = min(8, c1 - j);
        Raw8<T> r = {};
        if (base != nullptr) r = load8(base + (tl.t0 + t) * ldb + j, valid);
        store8(out + (tl.t0 + t) * ldo + j, r, valid);
      }
    return;
  }
  Frag<T, float> fh[NT][RK];
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int b = 0; b < RK; ++b) {
      const int t = u * 16 + n, i = b * 32 + g * 8;
      Raw8<float> h = {};
      if (t < tl.n) {
        const int64_t at = static_cast<int64_t>(tl.t0 + t) * rank + i;
        for (int p = 0; p < parts; ++p) {
          const Raw8<float> q = load8(H + p * sg.tokens * rank + at, rank - i);
#pragma unroll
          for (int e = 0; e < 8; ++e) h.v[e] += q.v[e];
        }
        if (Hsum != nullptr && blockIdx.y == 0 && wave == 0) store8(Hsum + at, h, rank - i);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) h.v[e] *= scale;
      fh[u][b] = frag_of<T, float>(h);
    }
  const W* wc = w + tl.slot * ldw;
  for (int j0 = c0 + wave * kExpandCols; j0 < c1; j0 += 4 * kExpandCols) {
    f32x4 acc[NT][8] = {};
#pragma unroll
    for (int b = 0; b < RK; ++b) {
      const int i = b * 32 + g * 8;
      if constexpr (AT) {
        // row q of product a is column j0 + (a / 2) * 32 + (q / 4) * 8 + (a % 2) * 4 + q % 4
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const int j = min(j0 + (a >> 1) * 32 + (n >> 2) * 8 + (a & 1) * 4 + (n & 3), width - 1);
          const Frag<T, W> fw = frag_of<T, W>(load8(wc + static_cast<int64_t>(j) * rank + i, rank - i));
#pragma unroll
          for (int u = 0; u < NT; ++u) mma(acc[u][a], fw, fh[u][b]);
        }
      } else {
        // row q of product a is column j0 + q * 8 + a: 8 loads of 8 columns hold 8 products' operands
        Frag<T, W> fw[8];
        const int j = j0 + n * 8, valid = max(0, min(8, width - j));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Raw8<W> r = load8(wc + static_cast<int64_t>(i + e) * width + j, i + e < rank ? valid : 0);
#pragma unroll
          for (int a = 0; a < 8; ++a) put_elem<T, W>(fw[a], e, r.v[a]);
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int u = 0; u < NT; ++u) mma(acc[u][a], fw[a], fh[u][b]);
      }
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int t = u * 16 + n;
      if (t >= tl.n) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = AT ? j0 + q * 32 + g * 8 : j0 + (g * 4 + q) * 8;
        const int valid = min(8, c1 - j);
        if (valid <= 0) continue;
        Raw8<T> r = {};
        if (base != nullptr) r = load8(base + (tl.t0 + t) * ldb + j, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          r.v[e] = from_f32<T>(to_f32(r.v[e]) + (AT ? acc[u][2 * q + (e >> 2)][e & 3] : acc[u][e][q]));
        store8(out + (tl.t0 + t) * ldo + j, r, valid);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// outer: G_c[i, j] = scale * sum over the tokens t of slot c of H[t, i] x[t, j].
// A workgroup takes one slot, 128 columns and every gridDim.z-th group of 32 of
// its tokens, the 4 waves in turn.  The inner index is the token: a lane loads
// 8 columns of each of its 8 tokens, which are the operands of 8 products with
// columns n * 8 + a.  With one part the sums go to G ([i][j], or [j][i] with AT),
// else each part's to its own copy (slot stride rank * width) for join_parts.
// ---------------------------------------------------------------------------
constexpr int kOuterCols = 128;

template <typename T, int RT, bool AT>
__global__ void __launch_bounds__(256)
    outer_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ H, Segs sg, int width, int rank,
                 float scale, float* __restrict__ G, int64_t ldg, int64_t part_stride, int accumulate) {
  __shared__ f32x4 sums[2][RT * 8][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int c = blockIdx.y, j = static_cast<int>(blockIdx.x) * kOuterCols + n * 8;
  const int valid = max(0, min(8, width - j));
  const int turns = 4 * static_cast<int>(gridDim.z), mine = static_cast<int>(blockIdx.z) * 4 + wave;
  f32x4 acc[RT][8] = {};
  int group = 0;
  bool any = false;
  for (int s0 = 0; s0 < sg.nseg; s0 += 64) {
    unsigned long long hits = __ballot(s0 + lane < sg.nseg && sg.slots[min(s0 + lane, sg.nseg - 1)] == c);
    for (; hits != 0; hits &= hits - 1) {
      const int s = s0 + __ffsll(hits) - 1;
      const int t0 = seg_start(sg, s + 1), t1 = seg_start(sg, s + 2);
      any |= t1 > t0;
      for (int t = t0; t < t1; t += 32, ++group) {
        if (group % turns != mine) continue;
        const int tg = t + g * 8, left = t1 - tg;          // tokens of other segments enter as zeros
        Frag<T, T> fx[8];
        Frag<T, float> fh[RT];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Raw8<T> r = load8(x + static_cast<int64_t>(min(tg + e, t1 - 1)) * ldx + j, e < left ? valid : 0);
#pragma unroll
          for (int a = 0; a < 8; ++a) put_elem<T, T>(fx[a], e, r.v[a]);
        }
#pragma unroll
        for (int b = 0; b < RT; ++b) {
          const int i = b * 16 + n;
          fh[b] = frag_of<T, float>(load8_strided(H + static_cast<int64_t>(tg) * rank + i, rank, i < rank ? left : 0));
        }
#pragma unroll
        for (int b = 0; b < RT; ++b)
#pragma unroll
          for (int a = 0; a < 8; ++a) mma(acc[b][a], fh[b], fx[a]);
      }
    }
  }
  // the waves' sums in a fixed order: (0 + 2) + (1 + 3)
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int q = 0; q < RT * 8; ++q) sums[wave - half][q][lane] = acc[q >> 3][q & 7];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int q = 0; q < RT * 8; ++q) acc[q >> 3][q & 7] += sums[wave][q][lane];
  }
  if (wave != 0 || (accumulate && !any && gridDim.z == 1)) return;
  const bool last = gridDim.z == 1;
  const bool add = last && accumulate;
  float* gc = G + blockIdx.z * part_stride + c * ldg;
  const float f = last ? scale : 1.f;
#pragma unroll
  for (int b = 0; b < RT; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = b * 16 + g * 4 + q;
      if (i >= rank) continue;
#pragma unroll
      for (int a = 0; a < 8; ++a) {
        if (a >= valid) continue;
        float* p = gc + (AT && last ? static_cast<int64_t>(j + a) * rank + i : static_cast<int64_t>(i) * width + j + a);
        const float v = f * acc[b][a][q];
        *p = add ? *p + v : v;
      }
    }
}

// G_c = scale * sum of the parts, in order
template <bool AT>
__global__ void __launch_bounds__(256)
    join_parts_kernel(const float* __restrict__ P, int parts, int64_t part_stride, Segs sg, int width, int rank,
                      float scale, float* __restrict__ G, int64_t ldg, int accumulate) {
  const int c = blockIdx.y;
  const int64_t per = static_cast<int64_t>(rank) * width;
  const int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (q >= per) return;
  if (accumulate) {
    bool any = false;
    for (int s = 0; s < sg.nseg; ++s) any |= sg.slots[s] == c && seg_start(sg, s + 2) > seg_start(sg, s + 1);
    if (!any) return;
  }
  const int64_t i = AT ? q % rank : q / width, j = AT ? q / rank : q % width;
  const float* p = P + c * per + i * width + j;
  float a = p[0];
  for (int z = 1; z < parts; ++z) a += p[z * part_stride];
  float* o = G + c * ldg + q;
  *o = accumulate ? *o + scale * a : scale * a;
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
  SRA_REQUIRE(sh.k >= 1 && sh.m >= 1 && sh.k < (int64_t{1} << 31) && sh.m < (int64_t{1} << 31), SRA_ERR_SHAPE,
              "k and m must be in [1, 2^31), got %lld, %lld", static_cast<long long>(sh.k),
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

// Parts of the width that shrink sums apart.  A tile's workgroup reads a whole
// client's weight, so with fewer tiles than compute units the width is split
// until there are enough workgroups, a part never below 512 columns.
static int shrink_parts(int64_t tokens, int64_t width) {
  int p = 1;
  while (p < kMaxParts && tokens * p < 64 && width >= 1024 * p) p *= 2;
  return p;
}

// Tokens per tile / 16: the most that still leaves a workgroup a compute unit.
static int tile_width(int64_t tokens) { return tokens >= 64 * 256 ? 4 : tokens >= 32 * 256 ? 2 : 1; }

// Parts of a client's tokens that outer sums apart: enough workgroups for the
// card, each with at least 8 groups of 32 tokens.
static int outer_parts(int64_t tokens, int64_t width, int nslots) {
  const int64_t blocks = cdiv(width, kOuterCols) * nslots;
  const int64_t groups = cdiv(tokens, 32 * static_cast<int64_t>(nslots));
  int p = 1;
  while (p < kMaxParts && blocks * p < 512 && groups >= 16 * p) p *= 2;
  return p;
}

struct Workspace {
  size_t h, z, ga, gb, bytes;
};

static Workspace plan(int64_t tokens, int64_t k, int64_t m, int rank, int nslots) {
  const size_t row = static_cast<size_t>(rank) * 4;
  const int pa = outer_parts(tokens, k, nslots), pb = outer_parts(tokens, m, nslots);
  Workspace w{};
  w.h = 0;
  w.z = w.h + static_cast<size_t>(tokens) * row * shrink_parts(tokens, k);
  w.ga = w.z + static_cast<size_t>(tokens) * row * (shrink_parts(tokens, m) + 1);
  w.gb = w.ga + (pa > 1 ? static_cast<size_t>(pa) * nslots * k * row : 0);
  w.bytes = w.gb + (pb > 1 ? static_cast<size_t>(pb) * nslots * m * row : 0) + 16;
  return w;
}

template <typename F>
static int with_tile(int64_t tokens, F&& f) {
  switch (tile_width(tokens)) {
    case 4: return f(std::integral_constant<int, 4>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 1>{});
  }
}

template <typename T, typename W, bool AT>
static int launch_shrink(const void* x, int64_t ldx, const void* w, int64_t ldw, const Segs& sg, int64_t width,
                         int parts, int rank, float* H, hipStream_t st) {
  const int part = static_cast<int>(cdiv(cdiv(width, parts), 32) * 32);
  return with_tile(sg.tokens, [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    hipLaunchKernelGGL((shrink_kernel<T, W, NT, AT>), dim3(tile_count<16 * NT>(sg), parts), dim3(kShrinkWaves * 64),
                       0, st, static_cast<const T*>(x), ldx, static_cast<const W*>(w), ldw, sg,
                       static_cast<int>(width), part, rank, H);
    return launch_status("shrink_kernel");
  });
}

template <typename T, typename W, bool AT>
static int launch_expand(const void* base, int64_t ldb, const float* H, int parts, const void* w, int64_t ldw,
                         const Segs& sg, int64_t width, int rank, float scale, void* out, int64_t ldo, float* Hsum,
                         hipStream_t st) {
  return with_tile(sg.tokens, [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    const int tiles = tile_count<16 * NT>(sg);
    // at least 2048 workgroups where the width allows it
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(cdiv(2048, tiles), cdiv(width, 4 * kExpandCols)));
    const int span = static_cast<int>(cdiv(cdiv(width, blocks), 4 * kExpandCols) * 4 * kExpandCols);
    const dim3 grid(tiles, static_cast<unsigned>(cdiv(width, span)));
    auto go = [&](auto rk) {
      constexpr int RK = decltype(rk)::value;
      hipLaunchKernelGGL((expand_kernel<T, W, RK, NT, AT>), grid, dim3(256), 0, st, static_cast<const T*>(base), ldb,
                         H, parts, static_cast<const W*>(w), ldw, sg, static_cast<int>(width), span, rank, scale,
                         static_cast<T*>(out), ldo, Hsum);
      return launch_status("expand_kernel");
    };
    return rank <= 32 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
  });
}

template <typename T, bool AT>
static int launch_outer(const void* x, int64_t ldx, const float* H, const Segs& sg, int64_t width, int rank,
                        float scale, float* G, int64_t ldg, int accumulate, float* parts_ws, hipStream_t st) {
  const int parts = outer_parts(sg.tokens, width, sg.nslots);
  const int64_t per = rank * width, stride = per * sg.nslots;
  const dim3 grid(static_cast<unsigned>(cdiv(width, kOuterCols)), static_cast<unsigned>(sg.nslots), parts);
  auto go = [&](auto rt) {
    constexpr int RT = decltype(rt)::value;
    hipLaunchKernelGGL((outer_kernel<T, RT, AT>), grid, dim3(256), 0, st, static_cast<const T*>(x), ldx, H, sg,
                       static_cast<int>(width), rank, scale, parts > 1 ? parts_ws : G, parts > 1 ? per : ldg, stride,
                       accumulate);
    return launch_status("outer_kernel");
  };
  const int rc = rank <= 16 ? go(std::integral_constant<int, 1>{})
                            : rank <= 32 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 4>{});
  if (rc || parts == 1) return rc;
  const dim3 jg(static_cast<unsigned>(cdiv(per, 256)), static_cast<unsigned>(sg.nslots));
  hipLaunchKernelGGL((join_parts_kernel<AT>), jg, dim3(256), 0, st, parts_ws, parts, stride, sg,
                     static_cast<int>(width), rank, scale, G, ldg, accumulate);
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
  const int parts = shrink_parts(sg.tokens, sh.k);
  float* H = parts == 1 && hidden != nullptr ? hidden : reinterpret_cast<float*>(ws);
  if (int rc = launch_shrink<T, W, false>(x, ldx, w.A, w.lda, sg, sh.k, parts, sh.rank, H, st)) return rc;
  return launch_expand<T, W, true>(base, ldbase, H, parts, w.B, w.ldb, sg, sh.m, sh.rank, sh.scale, out, ldo,
                                   parts > 1 ? hidden : nullptr, st);
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
      const int parts = g.dx != nullptr ? shrink_parts(sg.tokens, sh.m) : 1;
      float* Zp = Z;
      if (parts > 1) Z = Zp + static_cast<int64_t>(parts) * sg.tokens * sh.rank;
      if (int rc = launch_shrink<T, W, true>(dout, lddo, w.B, w.ldb, sg, sh.m, parts, sh.rank, Zp, st)) return rc;
      if (g.dx != nullptr)
        if (int rc = launch_expand<T, W, false>(g.dxbase, g.lddxb, Zp, parts, w.A, w.lda, sg, sh.k, sh.rank, sh.scale,
                                                g.dx, g.lddx, parts > 1 ? Z : nullptr, st))
          return rc;
    }
    if (g.dB != nullptr && H == nullptr) {
      H = Hw;
      if (int rc = launch_shrink<T, W, false>(x, ldx, w.A, w.lda, sg, sh.k, 1, sh.rank, Hw, st)) return rc;
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

extern "C" int sra_adapter_workspace_bytes(int64_t tokens, int64_t k, int64_t m, int32_t rank, int32_t nslots,
                                           size_t* bytes) {
  SRA_REQUIRE(bytes != nullptr, SRA_ERR_ARG, "null bytes pointer");
  if (int rc = check_tokens(tokens, nslots)) return rc;
  SRA_REQUIRE(k >= 1 && m >= 1, SRA_ERR_SHAPE, "k and m must be >= 1");
  SRA_REQUIRE(rank >= 1, SRA_ERR_ARG, "rank must be >= 1, got %d", rank);
  SRA_REQUIRE(rank <= SRA_ADAPTER_MAX_RANK, SRA_ERR_UNSUPPORTED, "rank %d is above %d", rank,
              SRA_ADAPTER_MAX_RANK);
  *bytes = plan(tokens, k, m, rank, nslots).bytes;
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
  if (int rc = sra_adapter_workspace_bytes(tokens, k, m, rank, nslots, &need)) return rc;
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
  if (int rc = sra_adapter_workspace_bytes(tokens, k, m, rank, nslots, &need)) return rc;
  SRA_REQUIRE(ws != nullptr && ws_bytes >= need, SRA_ERR_WORKSPACE, "adapter workspace: need %zu bytes, got %zu", need,
              ws_bytes);
  const GradOut g{hidden, dxbase, lddxb, dx, lddx, dA, ldda, dB, lddb, accumulate};
  const Weights wt{A, lda, B, ldb};
  return with_types(dtype, wdtype, [&](auto t, auto w) {
    return run_grad<decltype(t), decltype(w)>(dout, lddo, x, ldx, wt, sg, sh, g, static_cast<char*>(ws),
                                              plan(tokens, k, m, rank, nslots), static_cast<hipStream_t>(stream));
  });
}

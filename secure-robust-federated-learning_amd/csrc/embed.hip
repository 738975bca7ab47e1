// k13 — embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out_t = scale * E_c[ids[t]],   dE_c[v] = scale * sum_{t of c, ids[t] = v} dout_t
//
// The gradient sorts the tokens by (slot, id, position) and sums each run of
// equal rows in that order: no float atomics, so the result does not depend on
// the order in which workgroups run.
#include <algorithm>

#include "lm_common.hpp"

namespace sra {

unsigned int embed_row_faults(bool reset) { return tu_row_faults(reset); }

struct Tokens {
  const int64_t* ids;
  const int64_t* offsets;
  const int32_t* slots;
  int nseg, nslots;
  int64_t tokens, vocab, dim;
};

// row of the (nslots * vocab, dim) table that token t reads, -1 for none; one
// caller a token counts its fault
__device__ __forceinline__ int64_t token_row(const Tokens& k, int64_t t, int& slot, int64_t& id, bool count) {
  slot = token_slot(k.offsets, k.slots, k.nseg, k.nslots, t, count);
  id = k.ids[t];
  if (slot < 0) return -1;
  if (id < 0 || id >= k.vocab) {
    if (count) count_row_fault();
    return -1;
  }
  return slot * k.vocab + id;
}

// float32 product, then one rounding.  The compiler would fuse an fp16 operand's
// conversion with the product (and the product with the rounding to fp16),
// which rounds differently; the empty statement keeps the three apart.
__device__ __forceinline__ float scaled(float v, float scale) {
  asm volatile("" : "+v"(v));
  float r = v * scale;
  asm volatile("" : "+v"(r));
  return r;
}

// 8 consecutive values of a row at any alignment of their type (the hardware's
// global accesses take it)
typedef u32x4 __attribute__((aligned(2))) any_u32x4;

template <typename S>
struct Row8 {
  u32x4 v[sizeof(S) / 2];
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(S) == 4) {
      const unsigned word = v[e / 4][e % 4];
      return __builtin_bit_cast(float, word);
    } else {
      return to_f32(__builtin_bit_cast(S, static_cast<unsigned short>(v[0][e / 2] >> (e % 2 * 16))));
    }
  }
};

template <typename S>
__device__ __forceinline__ Row8<S> load8(const S* p) {
  Row8<S> r;
#pragma unroll
  for (int b = 0; b < static_cast<int>(sizeof(S) / 2); ++b) r.v[b] = reinterpret_cast<const any_u32x4*>(p)[b];
  return r;
}

template <typename S>
__device__ __forceinline__ void store8(S* p, const float (&x)[8]) {
  union {
    u32x4 v[sizeof(S) / 2];
    S s[8];
  } q;
#pragma unroll
  for (int e = 0; e < 8; ++e) q.s[e] = from_f32<S>(x[e]);
#pragma unroll
  for (int b = 0; b < static_cast<int>(sizeof(S) / 2); ++b) reinterpret_cast<any_u32x4*>(p)[b] = q.v[b];
}

// Lookup: LANES lanes a token, 8 values a lane and step.  Bound by memory (a
// read of the row, a write of the output); 16 lanes keep every lane busy at odd
// widths, 64 spread few tokens over more waves.  32768 tokens, 2048 float32 values
// to bf16: 59 us for 81 MB of different rows, some of them fetched by several dies
// (150 MB in all), and 134 MB written: 4.8 TB/s.
template <typename W, typename T, int LANES>
__global__ void __launch_bounds__(256) embed_kernel(const W* __restrict__ table, int64_t ldt, Tokens k, float scale,
                                                    T* __restrict__ out, int64_t ldo) {
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
  if (t >= k.tokens) return;
  const int first = static_cast<int>(threadIdx.x % LANES) * 8;
  int slot;
  int64_t id;
  const bool none = token_row(k, t, slot, id, first == 0) < 0;
  const int dim = static_cast<int>(k.dim);
  const W* src = table + (none ? 0 : slot * ldt + id * k.dim);
  T* dst = out + t * ldo;
#pragma unroll 4
  for (int j = first; j < dim; j += LANES * 8) {
    if (j + 8 <= dim) {
      const Row8<W> r = load8(src + j);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = none ? 0.f : scaled(r.get(e), scale);
      store8(dst + j, x);
    } else {
      for (int e = j; e < dim; ++e) dst[e] = from_f32<T>(none ? 0.f : scaled(to_f32(src[e]), scale));
    }
  }
}

// ---------------------------------------------------------------------------
// Sort: key = row << 32 | position, unique, so any correct sort is stable.
// Tokens without a row get the largest row and stay behind.  Tiles of 4096 are
// sorted in LDS: runs of 1, 2, 4, ... merged by rank, an element moving to its
// place in its own run plus the count of smaller ones in the partner run, each
// thread's 4 searches in step.  The same launch clears the gradient with the
// workgroups behind the sorting ones: the sort hides behind that write (32768
// tokens and 410 MB: 56 us, 7.3 TB/s).
// ---------------------------------------------------------------------------
constexpr int kTile = 4096;
constexpr int kSortThreads = 1024;
constexpr int kOwn = kTile / kSortThreads;
constexpr unsigned kNoRow = 0xffffffffu;

struct Clear {
  float* grad;
  int64_t ldg, per;          // floats of a slot
  int blocks;                // workgroups a slot
};

__device__ __forceinline__ void clear_rows(const Clear& z, int64_t block) {
  float* g = z.grad + block / z.blocks * z.ldg;
  const int64_t stride = static_cast<int64_t>(z.blocks) * kSortThreads * 4;
  for (int64_t i = (block % z.blocks * kSortThreads + threadIdx.x) * 4; i < z.per; i += stride) {
    if (i + 4 <= z.per) {
      reinterpret_cast<any_u32x4*>(g + i)[0] = u32x4{0, 0, 0, 0};
    } else {
      for (int64_t e = i; e < z.per; ++e) g[e] = 0.f;
    }
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_tiles_kernel(Tokens k, int64_t padding, int tiles,
                                                                  uint64_t* __restrict__ keys, Clear clear) {
  __shared__ uint64_t buf[2][kTile];
  if (static_cast<int>(blockIdx.x) >= tiles) {
    clear_rows(clear, static_cast<int64_t>(blockIdx.x) - tiles);
    return;
  }
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int n = static_cast<int>(min(static_cast<int64_t>(kTile), k.tokens - t0));
  int top = 1;
  while (top < n) top <<= 1;
  for (int i = threadIdx.x; i < top; i += kSortThreads) {
    unsigned row = kNoRow;
    if (i < n) {
      int slot;
      int64_t id;
      const int64_t r = token_row(k, t0 + i, slot, id, true);
      if (r >= 0 && id != padding) row = static_cast<unsigned>(r);
    }
    buf[0][i] = static_cast<uint64_t>(row) << 32 | static_cast<uint32_t>(t0 + i);
  }
  __syncthreads();
  int cur = 0;
  for (int len = 1; len < top; len <<= 1) {
    uint64_t key[kOwn];
    int at[kOwn], to[kOwn];
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
      const int i = min(q * kSortThreads + static_cast<int>(threadIdx.x), top - 1);
      key[q] = buf[cur][i];
      at[q] = (i & ~(len - 1)) ^ len;                                  // the partner run
      to[q] = (i & ~(2 * len - 1)) + (i & (len - 1)) - at[q];          // place, less what `at` counts from
    }
    // lower bound in len sorted keys: halve, then one last comparison
    for (int step = len >> 1; step > 0; step >>= 1)
#pragma unroll
      for (int q = 0; q < kOwn; ++q)
        if (buf[cur][at[q] + step - 1] < key[q]) at[q] += step;
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
      if (buf[cur][at[q]] < key[q]) ++at[q];
      if (q * kSortThreads + static_cast<int>(threadIdx.x) < top) buf[cur ^ 1][at[q] + to[q]] = key[q];
    }
    cur ^= 1;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys[t0 + i] = buf[cur][i];
}

// Sorted runs, kGroup neighbours into one: an element's place is its place in its
// own run plus the count of smaller elements of the other runs, 4 searches in
// step.  More runs than a group take more passes: all against all would cost
// their square.  8 runs of 4096: 18 us, a chain of 24 dependent reads.
// ---------------------------------------------------------------------------
constexpr int kGroup = 16;

__global__ void __launch_bounds__(256) merge_runs_kernel(const uint64_t* __restrict__ keys, int64_t tokens,
                                                         int64_t run, uint64_t* __restrict__ sorted) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens) return;
  const uint64_t key = keys[i];
  const int64_t mine = i / run, first = mine / kGroup * kGroup;
  const int64_t end = min(first + kGroup, (tokens + run - 1) / run);
  int64_t place = first * run + i - mine * run;
  for (int64_t q0 = first; q0 < end; q0 += 4) {
    int64_t at[4], from[4], n[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      from[q] = at[q] = min(q0 + q, end - 1) * run;
      const bool search = q0 + q < end && q0 + q != mine;
      n[q] = search ? min(run, tokens - at[q]) : 0;
    }
    // keys at and beyond n count as larger
    for (int64_t step = run / 2; step > 0; step >>= 1)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t probe = at[q] + step - 1;
        const bool in = probe - from[q] < n[q];
        if (in && keys[in ? probe : from[q]] < key) at[q] += step;
      }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool in = at[q] - from[q] < n[q];
      if (in && keys[in ? at[q] : from[q]] < key) ++at[q];
      place += at[q] - from[q];
    }
  }
  sorted[place] = key;
}

// ---------------------------------------------------------------------------
// Sum: a wave takes a window of sorted positions and 512 columns, 8 rows' loads in
// flight.  Runs that lie inside the window go to their row; a run that the window
// shares with the one before (head) or after (tail) leaves a partial sum.  The window
// where such a run starts then adds up the partials in order, one wave for 512
// columns: a run of most of a large batch (padding ids that padding_idx does not
// leave out) is bound by that (2^20 tokens x 512 bf16: spread over 50001 rows 0.90
// ms, half of them one id 3.3 ms, all of them 5.4 ms; left out by padding_idx 0.30).
// Bound by the gather of dout's rows: 32768 x 2048 bf16 75 us, the join 15 us.
// ---------------------------------------------------------------------------
constexpr int kBatch = 8;
constexpr int kCols = 512;

__device__ __forceinline__ unsigned row_at(const uint64_t* __restrict__ sorted, int64_t i) {
  return static_cast<unsigned>(sorted[i] >> 32);
}

// Positions a window: 32 (a partial sum for 32 rows read), fewer where the waves
// would not fill the card.  Added to a gradient, so without the clear, but with sort,
// merge and join, common ids first: 32768 x 2048 of 50001 rows 138 us, 162 us with 8;
// 2000 x 512 of 4001 36 us, 65 us with 32.
static int window_of(int64_t tokens, int64_t dim) {
  int w = 32;
  while (w > 8 && cdiv(tokens, w) * cdiv(dim, kCols) < 4096) w /= 2;
  return w;
}

struct Grad {
  float* grad;
  int64_t ldg;
  float scale;
  int accumulate;
};

__device__ __forceinline__ void put_cols(float* p, const float (&a)[8], int valid) {
  if (valid >= 8) {
    store8(p, a);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) p[e] = a[e];
  }
}

__device__ __forceinline__ void put_row(const Grad& o, const Tokens& k, unsigned row, int j, const float (&a)[8],
                                        int valid) {
  const unsigned vocab = static_cast<unsigned>(k.vocab), slot = row / vocab, id = row % vocab;
  float* g = o.grad + static_cast<int64_t>(slot) * o.ldg + static_cast<int64_t>(id) * k.dim + j;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = a[e] * o.scale;
  if (o.accumulate)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) v[e] += g[e];
  put_cols(g, v, valid);
}

// WIDE: rows of at least 8 values, read 8 at a time; lanes whose 8 would pass the
// end of the row read the last 8 and use their upper ones
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) sum_windows_kernel(const T* __restrict__ dout, int64_t lddo, Tokens k,
                                                          const uint64_t* __restrict__ sorted, Grad o, int window,
                                                          int chunks, int64_t units, float* __restrict__ head,
                                                          float* __restrict__ tail) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t w = unit / chunks, from = w * window, to = min(from + window, k.tokens);
  const int dim = static_cast<int>(k.dim);
  const int j = static_cast<int>(unit % chunks) * kCols + static_cast<int>(threadIdx.x & 63) * 8;
  if (j >= dim) return;
  const int valid = min(8, dim - j), shift = WIDE ? 8 - valid : 0;
  float a[8] = {};
  unsigned row = row_at(sorted, from);
  bool shared_front = from > 0 && row_at(sorted, from - 1) == row;
  for (int64_t i0 = from; i0 < to && row != kNoRow; i0 += kBatch) {
    Row8<T> r[kBatch];
    uint64_t key[kBatch + 1];
#pragma unroll
    for (int q = 0; q <= kBatch; ++q) key[q] = i0 + q < k.tokens ? sorted[i0 + q] : ~uint64_t{0};
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const T* p = dout + static_cast<int64_t>(static_cast<uint32_t>(key[i0 + q < to ? q : 0])) * lddo + j;
      if constexpr (WIDE) {
        r[q] = load8(p - shift);
      } else {
        union {
          Row8<T> r;
          T t[8];
        } u = {};
        for (int e = 0; e < valid; ++e) u.t[e] = p[e];
        r[q] = u.r;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (i0 + q >= to || row == kNoRow) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] += r[q].get(e);
      const unsigned next = static_cast<unsigned>(key[q + 1] >> 32);
      const bool end = i0 + q + 1 == to;
      if (next == row && !end) continue;
      if (WIDE && shift != 0) {                              // the upper values belong to this lane's columns
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[e] = 0.f;
#pragma unroll
          for (int f = e; f < 8; ++f)
            if (f - e == shift) u[e] = a[f];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = u[e];
      }
      if (shared_front) put_cols(head + w * k.dim + j, a, valid);    // also when it goes on behind the window
      else if (end && next == row && to < k.tokens) put_cols(tail + w * k.dim + j, a, valid);
      else put_row(o, k, row, j, a, valid);
      shared_front = false;
      row = next;
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = 0.f;
    }
  }
}

__global__ void __launch_bounds__(256) join_windows_kernel(Tokens k, const uint64_t* __restrict__ sorted, Grad o,
                                                           int window, int chunks, int64_t units, const float* __restrict__ head,
                                                           const float* __restrict__ tail) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t w = unit / chunks, from = w * window, to = from + window;
  const int dim = static_cast<int>(k.dim);
  const int j = static_cast<int>(unit % chunks) * kCols + static_cast<int>(threadIdx.x & 63) * 8;
  if (to >= k.tokens) return;
  const unsigned row = row_at(sorted, to - 1);
  if (row == kNoRow || row_at(sorted, to) != row) return;                       // nothing goes on
  if (from > 0 && row_at(sorted, from - 1) == row) return;                      // started further to the front
  // how many windows the run goes on for, 64 at a time
  int64_t last = w + 1;
  for (const int64_t windows = (k.tokens + window - 1) / window;; last += 64) {
    const int64_t v = last + static_cast<int64_t>(threadIdx.x & 63);
    const unsigned long long on = __ballot(v < windows && row_at(sorted, min(v, windows - 1) * window) == row);
    if (~on != 0) {
      last += __ffsll(~on) - 1;
      break;
    }
  }
  if (j >= dim) return;                                                        // every lane was needed above
  const int valid = min(8, dim - j);
  float a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = e < valid ? tail[w * k.dim + j + e] : 0.f;
  for (int64_t v0 = w + 1; v0 < last; v0 += kBatch) {
    float h[kBatch][8];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const float* p = head + min(v0 + q, last - 1) * k.dim + j;
      if (valid == 8) {
        const Row8<float> r = load8(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[q][e] = r.get(e);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[q][e] = e < valid ? p[e] : 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (v0 + q < last)
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += h[q][e];
  }
  put_row(o, k, row, j, a, valid);
}

static int check_table(const Tokens& k, int64_t ldt) {
  if (int rc = check_tokens(k.tokens, k.nslots)) return rc;
  SRA_REQUIRE(k.vocab >= 1 && k.dim >= 1 && k.dim < (int64_t{1} << 23) && k.vocab < (int64_t{1} << 31),
              SRA_ERR_SHAPE, "vocab must be in [1, 2^31) and dim in [1, 2^23), got %lld, %lld",
              static_cast<long long>(k.vocab), static_cast<long long>(k.dim));
  SRA_REQUIRE(k.nslots == 1 || ldt >= k.vocab * k.dim, SRA_ERR_SHAPE, "the slot stride must be >= vocab * dim");
  SRA_REQUIRE(k.tokens == 0 || k.ids != nullptr, SRA_ERR_ARG, "ids must be non-null");
  if (k.offsets == nullptr && k.slots == nullptr) {
    SRA_REQUIRE(k.nslots == 1, SRA_ERR_ARG, "tables of %d slots need offsets and slots", k.nslots);
    return SRA_OK;
  }
  return check_segments(k.offsets, k.slots, k.nseg);
}

struct GradPlan {
  size_t keys, sorted, head, tail, bytes;
};

static GradPlan grad_plan(int64_t tokens, int64_t dim) {
  GradPlan p{};
  const int64_t windows = cdiv(tokens, window_of(tokens, dim));
  p.keys = 0;
  p.sorted = p.keys + static_cast<size_t>(tokens) * 8;
  p.head = p.sorted + static_cast<size_t>(tokens) * 8;
  p.tail = p.head + static_cast<size_t>(windows) * dim * 4;
  p.bytes = p.tail + static_cast<size_t>(windows) * dim * 4 + 16;
  return p;
}

template <typename F>
static int with_type(int32_t dtype, F&& f) {
  if (dtype == SRA_F32) return f(float{});
  if (dtype == SRA_BF16) return f(__bf16{});
  return f(_Float16{});
}

}  // namespace sra

using namespace sra;

extern "C" int sra_embed(const void* table, int64_t ldt, int32_t tdtype, const int64_t* ids, const int64_t* offsets,
                         const int32_t* slots, int32_t nseg, int64_t tokens, int32_t nslots, int64_t vocab,
                         int64_t dim, float scale, void* out, int64_t ldo, int32_t odtype, void* stream) {
  const Tokens k{ids, offsets, slots, nseg, nslots, tokens, vocab, dim};
  if (int rc = check_table(k, ldt)) return rc;
  if (int rc = check_dtype(tdtype, "tdtype")) return rc;
  if (int rc = check_dtype(odtype, "odtype")) return rc;
  SRA_REQUIRE(table != nullptr && (out != nullptr || tokens == 0), SRA_ERR_ARG, "table and out must be non-null");
  SRA_REQUIRE(tokens <= 1 || ldo >= dim, SRA_ERR_SHAPE, "out needs a row stride >= dim");
  if (tokens == 0) return SRA_OK;
  return with_type(tdtype, [&](auto w) {
    return with_type(odtype, [&](auto t) -> int {
      using W = decltype(w);
      using T = decltype(t);
      // 16 lanes a token unless that leaves the card less than 4 waves a compute unit
      // (1024 values: 1000 tokens 7.2 us with 16 lanes, 4.4 with 64; 8000 9.9, 9.7;
      // 16000 16.5, 16.9)
      const bool few = tokens * 16 < 64 * 1024;
      const int64_t blocks = cdiv(tokens * (few ? 64 : 16), 256);
      if (int rc = check_launch(blocks, 256)) return rc;
      SRA_REQUIRE(out != table, SRA_ERR_ARG, "out must not be the table: other tokens read it");
      const dim3 grid(static_cast<unsigned>(blocks));
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const W*>(table),
                           ldt, k, scale, static_cast<T*>(out), ldo);
        return launch_status("embed_kernel");
      };
      return few ? go(embed_kernel<W, T, 64>) : go(embed_kernel<W, T, 16>);
    });
  });
}

extern "C" int sra_embed_grad_workspace_bytes(int64_t tokens, int64_t dim, size_t* bytes) {
  SRA_REQUIRE(bytes != nullptr, SRA_ERR_ARG, "null bytes pointer");
  if (int rc = check_tokens(tokens, 1)) return rc;
  SRA_REQUIRE(dim >= 1 && dim < (int64_t{1} << 23), SRA_ERR_SHAPE, "dim must be in [1, 2^23), got %lld",
              static_cast<long long>(dim));
  *bytes = grad_plan(tokens, dim).bytes;
  return SRA_OK;
}

extern "C" int sra_embed_grad(const void* dout, int64_t lddo, int32_t dtype, const int64_t* ids,
                              const int64_t* offsets, const int32_t* slots, int32_t nseg, int64_t tokens,
                              int32_t nslots, int64_t vocab, int64_t dim, float scale, int64_t padding, float* grad,
                              int64_t ldg, int32_t accumulate, void* ws, size_t ws_bytes, void* stream) {
  const Tokens k{ids, offsets, slots, nseg, nslots, tokens, vocab, dim};
  if (int rc = check_table(k, ldg)) return rc;
  if (int rc = check_dtype(dtype, "dtype")) return rc;
  SRA_REQUIRE(grad != nullptr && (dout != nullptr || tokens == 0), SRA_ERR_ARG, "dout and grad must be non-null");
  SRA_REQUIRE(tokens <= 1 || lddo >= dim, SRA_ERR_SHAPE, "dout needs a row stride >= dim");
  SRA_REQUIRE(static_cast<double>(nslots) * static_cast<double>(vocab) < 4294967295.0, SRA_ERR_UNSUPPORTED,
              "nslots * vocab must be below 2^32 - 1");
  const GradPlan p = grad_plan(tokens, dim);
  SRA_REQUIRE(ws != nullptr && ws_bytes >= p.bytes, SRA_ERR_WORKSPACE, "embed_grad workspace: need %zu bytes, got %zu",
              p.bytes, ws_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* base = static_cast<char*>(ws);
  uint64_t* keys = reinterpret_cast<uint64_t*>(base + p.keys);
  uint64_t* sorted = reinterpret_cast<uint64_t*>(base + p.sorted);
  float* head = reinterpret_cast<float*>(base + p.head);
  float* tail = reinterpret_cast<float*>(base + p.tail);
  const int tiles = static_cast<int>(cdiv(tokens, kTile));
  Clear clear{grad, ldg, vocab * dim, 0};
  if (!accumulate) {
    // one store a thread (983 MB: 156 us, against 172 us with 15 stores a thread),
    // more only where that would be too many workgroups for a launch (above 32 GiB)
    const int64_t most = cdiv(clear.per, kSortThreads * 4);
    clear.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (int64_t{1} << 21) / nslots)));
  }
  if (tiles == 0 && accumulate) return SRA_OK;
  const int64_t blocks = tiles + static_cast<int64_t>(clear.blocks) * nslots;
  if (int rc = check_launch(blocks, kSortThreads)) return rc;
  const int chunks = static_cast<int>(cdiv(dim, kCols));
  const int window = window_of(tokens, dim);
  const int64_t units = cdiv(tokens, window) * chunks;
  if (int rc = check_launch(cdiv(units, 4), 256)) return rc;
  SRA_REQUIRE(tokens == 0 || dout != grad, SRA_ERR_ARG, "grad must not be dout: it is written before dout is read");
  // the passes end in `sorted`
  int passes = 0;
  for (int64_t run = kTile; run < tokens; run *= kGroup) ++passes;
  uint64_t* src = passes % 2 ? keys : sorted;
  hipLaunchKernelGGL(sort_tiles_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kSortThreads), 0, st, k, padding,
                     tiles, src, clear);
  if (int rc = launch_status("sort_tiles_kernel")) return rc;
  if (tokens == 0) return SRA_OK;
  for (int64_t run = kTile; run < tokens; run *= kGroup) {
    uint64_t* dst = src == keys ? sorted : keys;
    hipLaunchKernelGGL(merge_runs_kernel, dim3(static_cast<unsigned>(cdiv(tokens, 256))), dim3(256), 0, st, src,
                       tokens, run, dst);
    if (int rc = launch_status("merge_runs_kernel")) return rc;
    src = dst;
  }
  const dim3 grid(static_cast<unsigned>(cdiv(units, 4)));
  const Grad o{grad, ldg, scale, accumulate};
  const int rc = with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, static_cast<const T*>(dout), lddo, k, sorted, o, window,
                         chunks, units, head, tail);
      return launch_status("sum_windows_kernel");
    };
    return dim >= 8 ? go(sum_windows_kernel<T, true>) : go(sum_windows_kernel<T, false>);
  });
  if (rc || tokens <= window) return rc;
  hipLaunchKernelGGL(join_windows_kernel, grid, dim3(256), 0, st, k, sorted, o, window, chunks, units, head,
                     tail);
  return launch_status("join_windows_kernel");
}

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

// row of the (nslots * vocab, dim) table that token t reads, -1 for none
__device__ __forceinline__ int64_t token_row(const Tokens& k, int64_t t, int& slot, int64_t& id) {
  slot = token_slot(k.offsets, k.slots, k.nseg, k.nslots, t);
  id = k.ids[t];
  if (slot < 0) return -1;
  if (id < 0 || id >= k.vocab) {
    count_row_fault();
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

template <typename W, typename T>
__global__ void __launch_bounds__(256) embed_kernel(const W* __restrict__ table, int64_t ldt, Tokens k, float scale,
                                                    T* __restrict__ out, int64_t ldo) {
  const int64_t t = blockIdx.x;
  __shared__ int64_t src;
  if (threadIdx.x == 0) {
    int slot;
    int64_t id;
    src = token_row(k, t, slot, id) < 0 ? -1 : slot * ldt + id * k.dim;
  }
  __syncthreads();
  const int64_t from = src;
  for (int64_t j = threadIdx.x; j < k.dim; j += 256)
    out[t * ldo + j] = from_f32<T>(from < 0 ? 0.f : scaled(to_f32(table[from + j]), scale));
}

// ---------------------------------------------------------------------------
// Sort: key = row << 32 | position, unique, so any correct sort is stable.
// Tokens without a row get the largest row and stay behind.
// ---------------------------------------------------------------------------
constexpr int kTile = 4096;
constexpr int kSortThreads = 1024;
constexpr unsigned kNoRow = 0xffffffffu;

__global__ void __launch_bounds__(kSortThreads) sort_tiles_kernel(Tokens k, int64_t padding,
                                                                  uint64_t* __restrict__ keys) {
  __shared__ uint64_t buf[2][kTile];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int n = static_cast<int>(min(static_cast<int64_t>(kTile), k.tokens - t0));
  for (int i = threadIdx.x; i < kTile; i += kSortThreads) {
    unsigned row = kNoRow;
    if (i < n) {
      int slot;
      int64_t id;
      const int64_t r = token_row(k, t0 + i, slot, id);
      if (r >= 0 && id != padding) row = static_cast<unsigned>(r);
    }
    buf[0][i] = static_cast<uint64_t>(row) << 32 | static_cast<uint32_t>(t0 + i);
  }
  __syncthreads();
  // runs of 1, 2, 4, ... merged by rank: an element moves to its place in its
  // own run plus the count of smaller ones in the partner run
  int cur = 0;
  int top = 1;
  while (top < n) top <<= 1;
  for (int len = 1; len < top; len <<= 1) {
    for (int i = threadIdx.x; i < top; i += kSortThreads) {
      const uint64_t key = buf[cur][i];
      const int mine = i & ~(len - 1), other = mine ^ len, base = mine & ~(2 * len - 1);
      int lo = 0, hi = len;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (buf[cur][other + mid] < key) lo = mid + 1; else hi = mid;
      }
      buf[cur ^ 1][base + (i - mine) + lo] = key;
    }
    cur ^= 1;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) keys[t0 + i] = buf[cur][i];
}

// Sorted tiles into one sorted list: an element's place is its place in its own
// tile plus the count of smaller elements of every other tile.
__global__ void __launch_bounds__(256) merge_tiles_kernel(const uint64_t* __restrict__ keys, int64_t tokens,
                                                          uint64_t* __restrict__ sorted) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens) return;
  const uint64_t key = keys[i];
  const int64_t mine = i / kTile;
  int64_t place = i - mine * kTile;
  for (int64_t q = 0; q * kTile < tokens; ++q) {
    if (q == mine) continue;
    int64_t lo = q * kTile, hi = min(lo + kTile, tokens);
    const int64_t from = lo;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < key) lo = mid + 1; else hi = mid;
    }
    place += lo - from;
  }
  sorted[place] = key;
}

__global__ void __launch_bounds__(256) fill_rows_kernel(float* __restrict__ grad, int64_t ldg, int64_t per_slot) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  float* g = grad + blockIdx.y * ldg;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < per_slot; i += stride) g[i] = 0.f;
}

// ---------------------------------------------------------------------------
// Sum: a workgroup takes kWindow sorted positions of 256 columns.  Runs that
// lie inside the window go to their row; a run that the window shares with the
// one before (head) or after (tail) leaves a partial sum.  The window where
// such a run starts then adds up the partials in order.
// ---------------------------------------------------------------------------
constexpr int kWindow = 32;

__device__ __forceinline__ unsigned row_at(const uint64_t* __restrict__ sorted, int64_t i) {
  return static_cast<unsigned>(sorted[i] >> 32);
}

__device__ __forceinline__ void put(float* grad, int64_t ldg, const Tokens& k, unsigned row, int64_t j, float v,
                                    int accumulate) {
  const int64_t slot = row / k.vocab, id = row % k.vocab;
  float* g = grad + slot * ldg + id * k.dim + j;
  *g = accumulate ? *g + v : v;
}

template <typename T>
__global__ void __launch_bounds__(256) sum_windows_kernel(const T* __restrict__ dout, int64_t lddo, Tokens k,
                                                          const uint64_t* __restrict__ sorted, float scale,
                                                          float* __restrict__ grad, int64_t ldg, int accumulate,
                                                          float* __restrict__ head, float* __restrict__ tail) {
  const int64_t w = blockIdx.x, from = w * kWindow, to = min(from + kWindow, k.tokens);
  const int64_t j = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x;
  if (j >= k.dim) return;
  float a = 0.f;
  bool shared_front = from > 0 && row_at(sorted, from - 1) == row_at(sorted, from);
  for (int64_t i = from; i < to; ++i) {
    const unsigned row = row_at(sorted, i);
    if (row == kNoRow) break;
    a += to_f32(dout[static_cast<int64_t>(static_cast<uint32_t>(sorted[i])) * lddo + j]);
    if (i + 1 < to && row_at(sorted, i + 1) == row) continue;
    const bool shared_back = i + 1 == to && to < k.tokens && row_at(sorted, to) == row;
    if (shared_front) head[w * k.dim + j] = a;            // also when it goes on behind the window
    else if (shared_back) tail[w * k.dim + j] = a;
    else put(grad, ldg, k, row, j, a * scale, accumulate);
    shared_front = false;
    a = 0.f;
  }
}

__global__ void __launch_bounds__(256) join_windows_kernel(Tokens k, const uint64_t* __restrict__ sorted, float scale,
                                                           float* __restrict__ grad, int64_t ldg, int accumulate,
                                                           const float* __restrict__ head,
                                                           const float* __restrict__ tail) {
  const int64_t w = blockIdx.x, from = w * kWindow, to = from + kWindow;
  const int64_t j = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x;
  if (j >= k.dim || to >= k.tokens) return;
  const unsigned row = row_at(sorted, to - 1);
  if (row == kNoRow || row_at(sorted, to) != row) return;                       // nothing goes on
  if (from > 0 && row_at(sorted, from - 1) == row) return;                      // started further to the front
  float a = tail[w * k.dim + j];
  for (int64_t v = w + 1; v * kWindow < k.tokens && row_at(sorted, v * kWindow) == row; ++v) a += head[v * k.dim + j];
  put(grad, ldg, k, row, j, a * scale, accumulate);
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
  const int64_t windows = cdiv(tokens, kWindow);
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
    return with_type(odtype, [&](auto t) {
      using W = decltype(w);
      using T = decltype(t);
      hipLaunchKernelGGL((embed_kernel<W, T>), dim3(static_cast<unsigned>(tokens)), dim3(256), 0,
                         static_cast<hipStream_t>(stream), static_cast<const W*>(table), ldt, k, scale,
                         static_cast<T*>(out), ldo);
      return launch_status("embed_kernel");
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
  if (!accumulate) {
    const int64_t per = vocab * dim;
    const unsigned gx = static_cast<unsigned>(std::min<int64_t>(cdiv(per, 256), 4096));
    for (int32_t c = 0; c < nslots; c += 65535) {
      const unsigned gy = static_cast<unsigned>(std::min<int32_t>(nslots - c, 65535));
      hipLaunchKernelGGL(fill_rows_kernel, dim3(gx, gy), dim3(256), 0, st, grad + c * ldg, ldg, per);
      if (int rc = launch_status("fill_rows_kernel")) return rc;
    }
  }
  if (tokens == 0) return SRA_OK;
  const int64_t tiles = cdiv(tokens, kTile);
  hipLaunchKernelGGL(sort_tiles_kernel, dim3(static_cast<unsigned>(tiles)), dim3(kSortThreads), 0, st, k, padding,
                     tiles > 1 ? keys : sorted);
  if (int rc = launch_status("sort_tiles_kernel")) return rc;
  if (tiles > 1) {
    hipLaunchKernelGGL(merge_tiles_kernel, dim3(static_cast<unsigned>(cdiv(tokens, 256))), dim3(256), 0, st, keys,
                       tokens, sorted);
    if (int rc = launch_status("merge_tiles_kernel")) return rc;
  }
  const dim3 grid(static_cast<unsigned>(cdiv(tokens, kWindow)), static_cast<unsigned>(cdiv(dim, 256)));
  const int rc = with_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((sum_windows_kernel<T>), grid, dim3(256), 0, st, static_cast<const T*>(dout), lddo, k, sorted,
                       scale, grad, ldg, accumulate, head, tail);
    return launch_status("sum_windows_kernel");
  });
  if (rc) return rc;
  if (tokens > kWindow) {
    hipLaunchKernelGGL(join_windows_kernel, grid, dim3(256), 0, st, k, sorted, scale, grad, ldg, accumulate, head,
                       tail);
    return launch_status("join_windows_kernel");
  }
  return SRA_OK;
}

// k12 — low-rank adapters of many clients beside a shared projection.
//
//   h_t = A_c x_t,  out_t = base_t + scale * B_c h_t          (c = slot of t)
//   z_t = B_c' dout_t,  dx_t = dxbase_t + scale * A_c' z_t
//   dA_c = scale * sum_t z_t x_t',  dB_c = scale * sum_t dout_t h_t'
//
// Both directions are the same three products with the roles of (x, A, B) and
// (dout, B', A') exchanged, so each kernel takes the weight as an element
// stride pair.
#include "lm_common.hpp"

namespace sra {

unsigned int adapter_row_faults(bool reset) { return tu_row_faults(reset); }

struct Segs {
  const int64_t* offsets;
  const int32_t* slots;
  int nseg, nslots;
  int64_t tokens;
};

// H[t, i] = sum_j W_c[i, j] x[t, j] over j < width: one workgroup a token.
template <typename T, typename W>
__global__ void __launch_bounds__(256) shrink_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w,
                                                     int64_t ldw, int64_t si, int64_t sj, Segs sg, int64_t width,
                                                     int rank, float* __restrict__ H) {
  const int64_t t = blockIdx.x;
  const int c = token_slot(sg.offsets, sg.slots, sg.nseg, sg.nslots, t);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = wave; i < rank; i += 4) {
    float a = 0.f;
    if (c >= 0) {
      for (int64_t j = lane; j < width; j += 64)
        a += to_f32(w[c * ldw + i * si + j * sj]) * to_f32(x[t * ldx + j]);
      for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o);
    }
    if (lane == 0) H[t * rank + i] = a;
  }
}

// out[t, j] = base[t, j] + scale * sum_i W_c[i, j] H[t, i].
template <typename T, typename W>
__global__ void __launch_bounds__(256) expand_kernel(const T* base, int64_t ldb, const float* __restrict__ H,
                                                     const W* __restrict__ w, int64_t ldw, int64_t si, int64_t sj,
                                                     Segs sg, int64_t width, int rank, float scale, T* out,
                                                     int64_t ldo) {
  const int64_t t = blockIdx.x;
  const int c = token_slot(sg.offsets, sg.slots, sg.nseg, sg.nslots, t);
  for (int64_t j = threadIdx.x; j < width; j += 256) {
    const float b = base != nullptr ? to_f32(base[t * ldb + j]) : 0.f;
    float a = 0.f;
    if (c >= 0)
      for (int i = 0; i < rank; ++i) a += to_f32(w[c * ldw + i * si + j * sj]) * H[t * rank + i];
    out[t * ldo + j] = from_f32<T>(c >= 0 ? b + scale * a : b);
  }
}

// G_c[i, j] (+)= scale * sum over the tokens t of slot c of H[t, i] x[t, j].
template <typename T>
__global__ void __launch_bounds__(256) outer_kernel(const T* __restrict__ x, int64_t ldx,
                                                    const float* __restrict__ H, Segs sg, int64_t width, int rank,
                                                    float scale, float* __restrict__ G, int64_t ldg, int64_t si,
                                                    int64_t sj, int accumulate) {
  const int c = blockIdx.y;
  const int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t j = q % width;
  const int i = static_cast<int>(q / width);
  if (i >= rank) return;
  float a = 0.f;
  for (int s = 0; s < sg.nseg; ++s) {
    if (sg.slots[s] != c) continue;
    const int64_t t0 = max(sg.offsets[s], int64_t{0}), t1 = min(sg.offsets[s + 1], sg.tokens);
    for (int64_t t = t0; t < t1; ++t) a += H[t * rank + i] * to_f32(x[t * ldx + j]);
  }
  float* g = G + c * ldg + i * si + j * sj;
  *g = accumulate ? *g + scale * a : scale * a;
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

static size_t hidden_bytes(int64_t tokens, int rank) { return static_cast<size_t>(tokens) * rank * 4; }

template <typename T, typename W>
static int run_apply(const void* base, int64_t ldbase, const void* x, int64_t ldx, const void* A, int64_t lda,
                     const void* B, int64_t ldb, const Segs& sg, const Shape& sh, void* out, int64_t ldo, float* H,
                     hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(sg.tokens));
  hipLaunchKernelGGL((shrink_kernel<T, W>), grid, dim3(256), 0, st, static_cast<const T*>(x), ldx,
                     static_cast<const W*>(A), lda, sh.k, int64_t{1}, sg, sh.k, sh.rank, H);
  if (int rc = launch_status("shrink_kernel")) return rc;
  hipLaunchKernelGGL((expand_kernel<T, W>), grid, dim3(256), 0, st, static_cast<const T*>(base), ldbase, H,
                     static_cast<const W*>(B), ldb, int64_t{1}, static_cast<int64_t>(sh.rank), sg, sh.m, sh.rank,
                     sh.scale, static_cast<T*>(out), ldo);
  return launch_status("expand_kernel");
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
static int run_grad(const void* dout, int64_t lddo, const void* x, int64_t ldx, const void* A, int64_t lda,
                    const void* B, int64_t ldb, const Segs& sg, const Shape& sh, const GradOut& g, float* Z, float* Hw,
                    hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(sg.tokens));
  const float* H = g.hidden;
  if (sg.tokens > 0) {
    if (g.dx != nullptr || g.dA != nullptr) {
      hipLaunchKernelGGL((shrink_kernel<T, W>), grid, dim3(256), 0, st, static_cast<const T*>(dout), lddo,
                         static_cast<const W*>(B), ldb, int64_t{1}, static_cast<int64_t>(sh.rank), sg, sh.m, sh.rank,
                         Z);
      if (int rc = launch_status("shrink_kernel")) return rc;
    }
    if (g.dB != nullptr && H == nullptr) {
      H = Hw;
      hipLaunchKernelGGL((shrink_kernel<T, W>), grid, dim3(256), 0, st, static_cast<const T*>(x), ldx,
                         static_cast<const W*>(A), lda, sh.k, int64_t{1}, sg, sh.k, sh.rank, Hw);
      if (int rc = launch_status("shrink_kernel")) return rc;
    }
    if (g.dx != nullptr) {
      hipLaunchKernelGGL((expand_kernel<T, W>), grid, dim3(256), 0, st, static_cast<const T*>(g.dxbase), g.lddxb, Z,
                         static_cast<const W*>(A), lda, sh.k, int64_t{1}, sg, sh.k, sh.rank, sh.scale,
                         static_cast<T*>(g.dx), g.lddx);
      if (int rc = launch_status("expand_kernel")) return rc;
    }
  }
  if (g.dA != nullptr) {
    const dim3 og(static_cast<unsigned>(cdiv(sh.k * sh.rank, 256)), static_cast<unsigned>(sg.nslots));
    hipLaunchKernelGGL((outer_kernel<T>), og, dim3(256), 0, st, static_cast<const T*>(x), ldx, Z, sg, sh.k, sh.rank,
                       sh.scale, g.dA, g.ldda, sh.k, int64_t{1}, g.accumulate);
    if (int rc = launch_status("outer_kernel")) return rc;
  }
  if (g.dB != nullptr) {
    const dim3 og(static_cast<unsigned>(cdiv(sh.m * sh.rank, 256)), static_cast<unsigned>(sg.nslots));
    hipLaunchKernelGGL((outer_kernel<T>), og, dim3(256), 0, st, static_cast<const T*>(dout), lddo, H, sg, sh.m,
                       sh.rank, sh.scale, g.dB, g.lddb, int64_t{1}, static_cast<int64_t>(sh.rank), g.accumulate);
    if (int rc = launch_status("outer_kernel")) return rc;
  }
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
  *bytes = 2 * hidden_bytes(tokens, rank) + 16;
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
  float* H = hidden != nullptr ? hidden : static_cast<float*>(ws);
  return with_types(dtype, wdtype, [&](auto t, auto w) {
    return run_apply<decltype(t), decltype(w)>(base, ldbase, x, ldx, A, lda, B, ldb, sg, sh, out, ldo, H,
                                               static_cast<hipStream_t>(stream));
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
  if (dx == nullptr && dA == nullptr && dB == nullptr) return SRA_OK;
  size_t need = 0;
  if (int rc = sra_adapter_workspace_bytes(tokens, k, m, rank, nslots, &need)) return rc;
  SRA_REQUIRE(ws != nullptr && ws_bytes >= need, SRA_ERR_WORKSPACE, "adapter workspace: need %zu bytes, got %zu", need,
              ws_bytes);
  const GradOut g{hidden, dxbase, lddxb, dx, lddx, dA, ldda, dB, lddb, accumulate};
  float* Z = static_cast<float*>(ws);
  float* Hw = Z + tokens * rank;
  return with_types(dtype, wdtype, [&](auto t, auto w) {
    return run_grad<decltype(t), decltype(w)>(dout, lddo, x, ldx, A, lda, B, ldb, sg, sh, g, Z, Hw,
                                              static_cast<hipStream_t>(stream));
  });
}

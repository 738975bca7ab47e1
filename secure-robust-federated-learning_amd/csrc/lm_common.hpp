// Shared by the operators of clients that are language models (k12-k14):
// element types, the segment table that maps tokens to clients, and the host
// checks of both.
#pragma once

#include "sra_common.hpp"

namespace sra {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// One rounding to nearest even at the end; everything before it is float.
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

// of `tokens` tokens; called by one lane for them
__device__ __forceinline__ void count_row_fault(unsigned tokens = 1) {
#ifdef SRA_DEVICE_ASSERT
  __builtin_trap();
#else
  atomicAdd(&g_row_faults, tokens);
#endif
}

// slots[s] for a token of segment s, checked: -1 for none.
__device__ __forceinline__ int checked_slot(const int32_t* __restrict__ slots, int s, int nslots, bool count) {
  const int c = slots[s];
  if (c < -1 || c >= nslots) {
    if (count) count_row_fault();
    return -1;
  }
  return c;
}

// The last segment whose start is <= t: empty segments before it share its
// start and are passed over.  -1 when t lies before the first start.
__device__ __forceinline__ int segment_of(const int64_t* __restrict__ offsets, int nseg, int64_t t) {
  int lo = -1, hi = nseg;                 // offsets[lo] <= t < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// Slot of token t, -1 for none (no covering segment, slot -1, or a bad slot); one
// caller a token and call counts its fault.
__device__ __forceinline__ int token_slot(const int64_t* __restrict__ offsets, const int32_t* __restrict__ slots,
                                          int nseg, int nslots, int64_t t, bool count) {
  if (offsets == nullptr) return 0;
  const int s = segment_of(offsets, nseg, t);
  if (s < 0 || t >= offsets[s + 1]) return -1;
  return checked_slot(slots, s, nslots, count);
}

inline int dtype_size(int32_t dtype) { return dtype == SRA_F32 ? 4 : 2; }

inline int check_dtype(int32_t dtype, const char* what) {
  SRA_REQUIRE(dtype == SRA_F32 || dtype == SRA_BF16 || dtype == SRA_F16, SRA_ERR_ARG,
              "%s must be SRA_F32, SRA_BF16 or SRA_F16, got %d", what, dtype);
  return SRA_OK;
}

// Rows beyond 2^31 would not fit the kernels' token indices.
inline int check_tokens(int64_t tokens, int32_t nslots) {
  SRA_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 31), SRA_ERR_SHAPE, "tokens must be in [0, 2^31), got %lld",
              static_cast<long long>(tokens));
  SRA_REQUIRE(nslots >= 1, SRA_ERR_SHAPE, "nslots must be >= 1, got %d", nslots);
  return SRA_OK;
}

inline int check_segments(const int64_t* offsets, const int32_t* slots, int32_t nseg) {
  SRA_REQUIRE(nseg >= 0 && nseg <= (1 << 24), SRA_ERR_ARG, "nseg must be in [0, 2^24], got %d", nseg);
  SRA_REQUIRE(offsets != nullptr && (slots != nullptr || nseg == 0), SRA_ERR_ARG,
              "offsets and slots must be non-null");
  return SRA_OK;
}

// A launch holds fewer than 2^32 threads a dimension.
inline int check_launch(int64_t blocks, int threads) {
  SRA_REQUIRE(blocks * threads < (int64_t{1} << 32), SRA_ERR_UNSUPPORTED,
              "%lld workgroups of %d threads are too many for one launch: split the rows",
              static_cast<long long>(blocks), threads);
  return SRA_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

unsigned int adapter_row_faults(bool reset);
unsigned int embed_row_faults(bool reset);
unsigned int logprob_row_faults(bool reset);

}  // namespace sra

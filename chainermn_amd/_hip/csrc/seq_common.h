// Shared helpers of the sequence-model kernels (embedding, dropout, RMS
// norm, linear attention): native 16-bit types, vectors of up to 16 bytes,
// dispatch over type and vector width.
#pragma once

#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/hip/HIPException.h>

namespace seq {

using bf16 = __bf16;
using fp16 = _Float16;

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// Elements of 16 bytes: what a lane reads and writes at once.
template <typename T>
constexpr int kWidth = 16 / sizeof(T);

// A vector at any element's address: rows of odd lengths are read by 16 bytes
// too (gfx950 reads global memory at any alignment).
template <typename T, int N>
struct anywhere {
  typedef vec<T, N> type __attribute__((aligned(sizeof(T))));
};

// The first n of N elements, 0 < n; zero behind them.
template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float (&r)[N], long n = N) {
  if (n >= N) {
    if constexpr (N * sizeof(T) > 16) {
      float a[N / 2], b[N / 2];
      load<T, N / 2>(p, a);
      load<T, N / 2>(p + N / 2, b);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        r[i] = a[i];
        r[i + N / 2] = b[i];
      }
    } else {
      const vec<T, N> v =
          *reinterpret_cast<const typename anywhere<T, N>::type*>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = float(v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = i < n ? float(p[i]) : 0.f;
  }
}

// Rounds to nearest even, the one rounding of a result held in 16 bits.
// ONCE: it is not read again soon, and passes the caches by.
template <typename T, int N, bool ONCE = false>
__device__ __forceinline__ void store(T* p, const float (&r)[N], long n = N) {
  if (n >= N) {
    if constexpr (N * sizeof(T) > 16) {
      float a[N / 2], b[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        a[i] = r[i];
        b[i] = r[i + N / 2];
      }
      store<T, N / 2, ONCE>(p, a);
      store<T, N / 2, ONCE>(p + N / 2, b);
    } else {
      vec<T, N> v;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = T(r[i]);
      auto* at = reinterpret_cast<typename anywhere<T, N>::type*>(p);
      if constexpr (ONCE) __builtin_nontemporal_store(v, at);
      else *at = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = T(r[i]);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Calls f(T()) with the native type of a scalar type.
template <typename F>
void dispatch(at::ScalarType t, const char* what, F f) {
  switch (t) {
    case at::kFloat: f(float()); break;
    case at::kBFloat16: f(bf16()); break;
    case at::kHalf: f(fp16()); break;
    default:
      TORCH_CHECK(false, what, ": float32, bfloat16 or float16, not ", t);
  }
}

// A launch has fewer than 2^32 threads.
static inline void check_grid(long blocks, long threads, const char* what) {
  TORCH_CHECK(blocks * threads < (1l << 32), what,
              ": more elements than a launch has threads for");
}

static inline hipStream_t stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

}  // namespace seq

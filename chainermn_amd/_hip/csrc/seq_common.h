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

template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = float(*p);
  } else if constexpr (N * sizeof(T) > 16) {
    float a[N / 2], b[N / 2];
    load<T, N / 2>(p, a);
    load<T, N / 2>(p + N / 2, b);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      r[i] = a[i];
      r[i + N / 2] = b[i];
    }
  } else {
    const vec<T, N> v = *reinterpret_cast<const vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = float(v[i]);
  }
}

// Rounds to nearest even, the one rounding of a result held in 16 bits.
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&r)[N]) {
  if constexpr (N == 1) {
    *p = T(r[0]);
  } else if constexpr (N * sizeof(T) > 16) {
    float a[N / 2], b[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      a[i] = r[i];
      b[i] = r[i + N / 2];
    }
    store<T, N / 2>(p, a);
    store<T, N / 2>(p + N / 2, b);
  } else {
    vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = T(r[i]);
    *reinterpret_cast<vec<T, N>*>(p) = v;
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// The widest vector (in elements, at most 16 bytes) at which rows of `dim`
// elements can be read from `p` with a row stride of `stride`.
static inline int vector_width(const void* p, long dim, long stride,
                               int size) {
  int n = 16 / size;
  while (n > 1 && (dim % n || stride % n ||
                   reinterpret_cast<uintptr_t>(p) % (n * size)))
    n /= 2;
  return n;
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

// Calls f(T(), std::integral_constant<int, N>()) for a vector width N.
template <typename F>
void dispatch_vec(at::ScalarType t, int n, const char* what, F f) {
  dispatch(t, what, [&](auto x) {
    using T = decltype(x);
    if constexpr (sizeof(T) == 2) {
      if (n == 8) return f(x, std::integral_constant<int, 8>());
    }
    if (n == 4) return f(x, std::integral_constant<int, 4>());
    if (n == 2) return f(x, std::integral_constant<int, 2>());
    f(x, std::integral_constant<int, 1>());
  });
}

static inline hipStream_t stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

}  // namespace seq

// Dropout from a counter-based generator: no mask is stored.
//
//   y_i = x_i / (1 - ratio) where word i of the stream >= ratio * 2^32, or 0
//
// The stream is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011).  Element i takes word i % 4 of
// block i / 4; the key is a 64-bit seed, the upper counter half a 64-bit
// call number.  The backward pass is the same map of the output's gradient
// with the same key.
//
// A dropped element is zero whatever it was, NaN and infinity too.
//
// Bound by memory: one read and one write of each element.  A 32 x 32 bit
// product is one instruction here, so ten rounds for four elements stay below
// that.  2^27 elements of bf16: 97 us, 5.6 TB/s (torch's copy reaches 4.9).

#include "seq_common.h"

namespace {

using namespace seq;

__device__ __forceinline__ void philox(unsigned c0, unsigned c1, unsigned c2,
                                       unsigned c3, unsigned k0, unsigned k1,
                                       unsigned (&out)[4]) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = 0xD2511F53ull * c0;
    const unsigned long long b = 0xCD9E8D57ull * c2;
    c0 = unsigned(b >> 32) ^ c1 ^ k0;
    c1 = unsigned(b);
    c2 = unsigned(a >> 32) ^ c3 ^ k1;
    c3 = unsigned(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0;
  out[1] = c1;
  out[2] = c2;
  out[3] = c3;
}

// A thread takes 8 elements, two blocks of the stream.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(
    const T* __restrict__ x, T* __restrict__ y, const long* __restrict__ key,
    long n, unsigned threshold, float scale) {
  const unsigned long seed = key[0], call = key[1];
  const long stride = gridDim.x * 256l * 8;
  for (long i = (blockIdx.x * 256l + threadIdx.x) * 8; i < n; i += stride) {
    float r[8];
    load<T, 8>(x + i, r, n - i);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned long block = (unsigned long)i / 4 + h;
      unsigned word[4];
      philox(unsigned(block), unsigned(block >> 32), unsigned(call),
             unsigned(call >> 32), unsigned(seed), unsigned(seed >> 32),
             word);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[4 * h + j] = word[j] >= threshold ? r[4 * h + j] * scale : 0.f;
    }
    store<T, 8, true>(y + i, r, n - i);
  }
}

__global__ void dropout_next_key_kernel(long* state, long* key, long shift) {
  key[0] = (long)((unsigned long)state[0] + (unsigned long)shift);
  key[1] = state[1];
  state[1] += 1;
}

bool is_key(const torch::Tensor& t) {
  return t.is_cuda() && t.scalar_type() == at::kLong && t.numel() == 2 &&
         t.is_contiguous();
}

}  // namespace

torch::Tensor dropout(torch::Tensor x, torch::Tensor key, long threshold,
                      double scale) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous(),
              "dropout: a contiguous GPU tensor");
  TORCH_CHECK(is_key(key) && key.device() == x.device(),
              "dropout: the key is two int64 on the tensor's GPU");
  TORCH_CHECK(threshold >= 0 && threshold < (1l << 32),
              "dropout: threshold outside of 32 bits");
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty_like(x);
  const long n = x.numel();
  if (n == 0) return y;
  long blocks = (n + 2047) / 2048;
  // the rest by strides of the grid (2^27 elements of bf16, both passes: 207
  // us; with a workgroup for every 2048, 218 us)
  if (blocks > 8192) blocks = 8192;
  dispatch(x.scalar_type(), "dropout", [&](auto t) {
    using T = decltype(t);
    dropout_kernel<T><<<dim3(blocks), dim3(256), 0, stream()>>>(
        (const T*)x.data_ptr(), (T*)y.data_ptr(), key.data_ptr<long>(), n,
        (unsigned)threshold, (float)scale);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return y;
}

torch::Tensor dropout_next_key(torch::Tensor state, long shift) {
  TORCH_CHECK(is_key(state), "dropout_next_key: two int64 on a GPU");
  const c10::DeviceGuard guard(state.device());
  auto key = torch::empty_like(state);
  state.unsafeGetTensorImpl()->bump_version();
  dropout_next_key_kernel<<<dim3(1), dim3(1), 0, stream()>>>(
      state.data_ptr<long>(), key.data_ptr<long>(), shift);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return key;
}

// Root-mean-square norm with the residual's addition.
//
//   h = x + residual            (rounded once where it is written)
//   y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps)
//
// and, with g = gy * w and xhat = h * rstd,
//
//   dh = rstd * (g - xhat * mean(g * xhat)) + gh,   dw = sum_rows gy * xhat.
//
// A row stays in registers: every input is read once and every output
// written once, which bounds all three kernels.  The sum is fp32 wherever it
// is used; the backward pass adds x and the residual again, since the rounded
// sum would leave its rounding in dw.  Sums and rstd are fp32.
//
// A row belongs to `tpr` threads, 2^n of them, of 16 elements each: a wave has
// a row of 1024 or several shorter ones, and no barrier.  (524288 rows of 64
// in bf16, both passes: 81 us; with a wave for each row, 360 us.)
//
// 32768 x 1024 in bf16 with a residual: forward 50 us, 5.3 TB/s, backward 65
// us, 5.2 TB/s, and 5 us for the last sum of dw.  e4m3 with groups of 128 of
// 16384 x 4096: 108 us, 4.3 TB/s; 64 x 1024: 6 us, a launch.

#include "seq_common.h"

namespace {

using namespace seq;

constexpr int kMaxDim = 16384;

// vectors of a row that a thread holds
template <typename T>
constexpr int kHeld = 16 / kWidth<T>;
template <typename T>
using Part = float[kHeld<T>][kWidth<T>];

// The sum over the row's threads, for all of them.  `lds` holds one float
// for each wave of the workgroup and is written again by the next call, so
// that calls alternate between two of them.
__device__ __forceinline__ float row_sum(float v, int tpr, float* lds) {
  if (tpr < 64) {
    for (int off = tpr >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
  }
  v = wave_sum(v);
  if (tpr > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    const int base = threadIdx.x / tpr * (tpr >> 6);
    v = 0.f;
    for (int i = 0; i < tpr >> 6; ++i) v += lds[base + i];
  }
  return v;
}

__device__ __forceinline__ float row_max(float v, int tpr, float* lds) {
  for (int off = (tpr < 64 ? tpr : 64) >> 1; off > 0; off >>= 1)
    v = fmaxf(v, __shfl_xor(v, off, 64));
  if (tpr > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    const int base = threadIdx.x / tpr * (tpr >> 6);
    for (int i = 0; i < tpr >> 6; ++i) v = fmaxf(v, lds[base + i]);
  }
  return v;
}

// A thread's part of the weight.
template <typename T>
__device__ __forceinline__ void load_weight(const void* w, bool w32, int dim,
                                            int t, int tpr,
                                            Part<T>& r) {
  constexpr int VE = kWidth<T>;
#pragma unroll
  for (int k = 0; k < kHeld<T>; ++k) {
    const int c = (k * tpr + t) * VE;
    if (c >= dim) continue;
    if (w32) load<float, VE>((const float*)w + c, r[k], dim - c);
    else load<T, VE>((const T*)w + c, r[k], dim - c);
  }
}

// A thread's part of a row, zero behind its end.
template <typename T>
__device__ __forceinline__ void load_row(const T* x, int dim, int t, int tpr,
                                         Part<T>& r) {
  constexpr int VE = kWidth<T>;
#pragma unroll
  for (int k = 0; k < kHeld<T>; ++k) {
    const int c = (k * tpr + t) * VE;
    if (c < dim) {
      load<T, VE>(x + c, r[k], dim - c);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) r[k][i] = 0.f;
    }
  }
}

// h of a row and its rstd; the sum is written to `sum` if there is one.
template <typename T>
__device__ __forceinline__ float read_row(
    const T* x, const T* res, T* sum, int dim, int t, int tpr, float eps,
    float* lds, Part<T>& h) {
  constexpr int VE = kWidth<T>;
  load_row<T>(x, dim, t, tpr, h);
  if (res) {
    Part<T> r;
    load_row<T>(res, dim, t, tpr, r);
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) h[k][i] += r[k][i];
      const int c = (k * tpr + t) * VE;
      if (c < dim) store<T, VE, true>(sum + c, h[k], dim - c);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < kHeld<T>; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) sq += h[k][i] * h[k][i];
  return rsqrtf(row_sum(sq, tpr, lds) / dim + eps);
}

template <typename T>
__global__ __launch_bounds__(1024) void rms_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ res,
    const void* __restrict__ w, bool w32, T* __restrict__ y,
    T* __restrict__ sum, float* __restrict__ rstd_out, long rows, int dim,
    long xs, long rs, int tpr, float eps) {
  constexpr int VE = kWidth<T>;
  __shared__ float lds[2][16];
  const int t = threadIdx.x % tpr, per = blockDim.x / tpr;
  Part<T> wt;
  load_weight<T>(w, w32, dim, t, tpr, wt);
  int turn = 0;
  for (long r0 = blockIdx.x * (long)per; r0 < rows;
       r0 += gridDim.x * (long)per, turn ^= 1) {
    long row = r0 + threadIdx.x / tpr;
    const bool on = row < rows;  // the others are at barriers and shuffles
    if (!on) row = rows - 1;
    Part<T> h;
    const float rstd = read_row<T>(
        x + row * xs, res ? res + row * rs : nullptr, sum + row * dim, dim, t,
        tpr, eps, lds[turn], h);
    if (!on) continue;
    if (rstd_out && t == 0) rstd_out[row] = rstd;
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      const int c = (k * tpr + t) * VE;
      if (c < dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i) h[k][i] = h[k][i] * rstd * wt[k][i];
        store<T, VE, true>(y + row * dim + c, h[k], dim - c);
      }
    }
  }
}

__device__ __forceinline__ float e4m3_scale(float amax) {
  const float s = amax / 448.f;
  return s > 0.f ? s : 1.f;  // a row of zeros
}

// Four values as e4m3 bytes, rounded to nearest even.
__device__ __forceinline__ unsigned to_e4m3(float a, float b, float c,
                                            float d) {
  const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, low, true);
}

template <int N>
__device__ __forceinline__ void store_e4m3(unsigned char* p, float scale,
                                           const float (&y)[N], int n) {
  float q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float v = y[i] / scale;
    // comparisons keep NaN
    q[i] = v > 448.f ? 448.f : v < -448.f ? -448.f : v;
  }
  vec<unsigned, N / 4> u;
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    u[i] = to_e4m3(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
  if (n >= N) {
    typedef vec<unsigned, N / 4> bytes __attribute__((aligned(1)));
    *reinterpret_cast<bytes*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (u[i / 4] >> (i % 4 * 8)) & 0xff;
  }
}

// y in e4m3 with a scale for each row (group = 0) or each `group` columns,
// 2^n of them that at most a row's threads and a wave hold: amax / 448.
template <typename T>
__global__ __launch_bounds__(1024) void rms_fp8_kernel(
    const T* __restrict__ x, const T* __restrict__ res,
    const void* __restrict__ w, bool w32, unsigned char* __restrict__ q,
    float* __restrict__ scales, T* __restrict__ sum, long rows, int dim,
    long xs, long rs, int tpr, float eps, int group) {
  constexpr int VE = kWidth<T>;
  __shared__ float lds[2][16];
  __shared__ float top[2][16];
  const int t = threadIdx.x % tpr, per = blockDim.x / tpr;
  Part<T> wt;
  load_weight<T>(w, w32, dim, t, tpr, wt);
  int turn = 0;
  for (long r0 = blockIdx.x * (long)per; r0 < rows;
       r0 += gridDim.x * (long)per, turn ^= 1) {
    long row = r0 + threadIdx.x / tpr;
    const bool on = row < rows;
    if (!on) row = rows - 1;
    Part<T> h;
    const float rstd = read_row<T>(
        x + row * xs, res ? res + row * rs : nullptr, sum + row * dim, dim, t,
        tpr, eps, lds[turn], h);
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      const int c = (k * tpr + t) * VE;
      float m = 0.f;
      if (c < dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          h[k][i] = h[k][i] * rstd * wt[k][i];
          m = fmaxf(m, fabsf(h[k][i]));
        }
      }
      if (group) {
        for (int off = group / VE / 2; off > 0; off >>= 1)
          m = fmaxf(m, __shfl_xor(m, off, 64));
        if (c < dim && on) {
          const float s = e4m3_scale(m);
          if (c % group == 0) scales[row * (dim / group) + c / group] = s;
          store_e4m3<VE>(q + row * dim + c, s, h[k], dim - c);
        }
      }
      amax = fmaxf(amax, m);
    }
    if (group) continue;
    const float s = e4m3_scale(row_max(amax, tpr, top[turn]));
    if (!on) continue;
    if (t == 0) scales[row] = s;
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      const int c = (k * tpr + t) * VE;
      if (c < dim) store_e4m3<VE>(q + row * dim + c, s, h[k], dim - c);
    }
  }
}

// dh of all rows, and the sum of gy * xhat over the workgroup's rows in
// part[workgroup]: a thread's columns are the same for each of its rows.
template <typename T>
__global__ __launch_bounds__(1024) void rms_bwd_kernel(
    const T* __restrict__ gy, const T* __restrict__ x,
    const T* __restrict__ res, const T* __restrict__ gh,
    const void* __restrict__ w, bool w32, const float* __restrict__ rstd_in,
    T* __restrict__ dh, float* __restrict__ part, long rows, int dim, long xs,
    long rs, int tpr) {
  extern __shared__ float cols[];  // [dim], where a workgroup has more rows
  constexpr int VE = kWidth<T>;
  __shared__ float lds[2][16];
  const int t = threadIdx.x % tpr, per = blockDim.x / tpr;
  Part<T> wt, dw;
  load_weight<T>(w, w32, dim, t, tpr, wt);
#pragma unroll
  for (int k = 0; k < kHeld<T>; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[k][i] = 0.f;
  int turn = 0;
  for (long r0 = blockIdx.x * (long)per; r0 < rows;
       r0 += gridDim.x * (long)per, turn ^= 1) {
    long row = r0 + threadIdx.x / tpr;
    const bool on = row < rows;
    if (!on) row = rows - 1;
    Part<T> g, xh, add;
    load_row<T>(gy + row * dim, dim, t, tpr, g);
    load_row<T>(x + row * xs, dim, t, tpr, xh);
    if (res) {
      Part<T> r;
      load_row<T>(res + row * rs, dim, t, tpr, r);
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) xh[k][i] += r[k][i];
    }
    if (gh) {
      load_row<T>(gh + row * dim, dim, t, tpr, add);
    } else {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) add[k][i] = 0.f;
    }
    const float rstd = rstd_in[row];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      if ((k * tpr + t) * VE >= dim || !on) continue;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        xh[k][i] *= rstd;
        dw[k][i] += g[k][i] * xh[k][i];
        g[k][i] *= wt[k][i];
        dot += g[k][i] * xh[k][i];
      }
    }
    const float mean = row_sum(dot, tpr, lds[turn]) / dim;
    if (!on) continue;
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      const int c = (k * tpr + t) * VE;
      if (c < dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          add[k][i] += rstd * (g[k][i] - xh[k][i] * mean);
        store<T, VE, true>(dh + row * dim + c, add[k], dim - c);
      }
    }
  }
  // rows of one wave, then those of several
  for (int off = tpr; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) dw[k][i] += __shfl_xor(dw[k][i], off, 64);
  const int unit = tpr < 64 ? 64 : tpr, units = blockDim.x / unit;
  float* out = part + blockIdx.x * (long)dim;
  if (units == 1) {
#pragma unroll
    for (int k = 0; k < kHeld<T>; ++k) {
      const int c = (k * tpr + t) * VE;
      if (c < dim) store<float, VE>(out + c, dw[k], dim - c);
    }
    return;
  }
  for (int p = 0; p < units; ++p) {  // one after another
    if (threadIdx.x / unit == p && threadIdx.x % unit < tpr) {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k) {
        const int c = (k * tpr + t) * VE;
        if (c < dim) {
          if (p > 0) {
            float a[VE];
            load<float, VE>(cols + c, a, dim - c);
#pragma unroll
            for (int i = 0; i < VE; ++i) dw[k][i] += a[i];
          }
          if (p + 1 == units) store<float, VE>(out + c, dw[k], dim - c);
          else store<float, VE>(cols + c, dw[k], dim - c);
        }
      }
    }
    __syncthreads();
  }
}

// dw: 16 columns of a workgroup, 16 threads for each.
template <typename W>
__global__ __launch_bounds__(256) void rms_dw_kernel(
    const float* __restrict__ part, W* __restrict__ dw, int parts, int dim) {
  __shared__ float lds[16][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15);
  const int r = threadIdx.x >> 4;
  float acc = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int p = r; p < parts; p += 16) acc += part[(long)p * dim + c];
  }
  lds[r][threadIdx.x & 15] = acc;
  __syncthreads();
  if (r != 0 || c >= dim) return;
  for (int i = 1; i < 16; ++i) acc += lds[i][threadIdx.x];
  dw[c] = W(acc);
}

struct Rows {
  long rows;
  int dim, tpr, block;
};

void check_matrix(const torch::Tensor& t, const torch::Tensor& like,
                  const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 2 &&
              t.sizes() == like.sizes() &&
              t.scalar_type() == like.scalar_type() &&
              (t.stride(1) == 1 || t.size(1) == 1),
              "rms_norm: ", what, " must be a matrix like x with contiguous "
              "rows on its GPU");
}

void check_weight(const torch::Tensor& w, const torch::Tensor& x) {
  TORCH_CHECK(w.is_cuda() && w.device() == x.device() && w.dim() == 1 &&
              w.size(0) == x.size(1) && w.is_contiguous() &&
              (w.scalar_type() == x.scalar_type() ||
               w.scalar_type() == at::kFloat),
              "rms_norm: the weight is a contiguous vector for the rows, of "
              "their type or float32, on their GPU");
}

Rows plan(long rows, long dim, int tpr = 1) {
  TORCH_CHECK(dim >= 1 && dim <= kMaxDim, "rms_norm: rows of 1 to ", kMaxDim,
              " elements, not ", dim);
  while (tpr * 16 < dim) tpr *= 2;
  return Rows{rows, (int)dim, tpr, tpr < 256 ? 256 : tpr};
}

int grid_of(const Rows& r, int most) {
  const long per = r.block / r.tpr;
  const long n = (r.rows + per - 1) / per;
  return int(n < most ? n : most);
}

}  // namespace

// (y, h, rstd): h is empty without a residual.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> rms_norm_fwd(
    torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> res,
    double eps) {
  check_matrix(x, x, "x");
  check_weight(w, x);
  const c10::DeviceGuard guard(x.device());
  const long rows = x.size(0), dim = x.size(1);
  if (res) check_matrix(*res, x, "the residual");
  const Rows r = plan(rows, dim);
  auto y = torch::empty({rows, dim}, x.options());
  auto h = torch::empty({res ? rows : 0, dim}, x.options());
  auto rstd = torch::empty({rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return {y, h, rstd};
  dispatch(x.scalar_type(), "rms_norm", [&](auto t) {
    using T = decltype(t);
    rms_fwd_kernel<T>
        <<<dim3(grid_of(r, 4096)), dim3(r.block), 0, stream()>>>(
            (const T*)x.data_ptr(), res ? (const T*)res->data_ptr() : nullptr,
            w.data_ptr(), w.scalar_type() == at::kFloat, (T*)y.data_ptr(),
            (T*)h.data_ptr(), rstd.data_ptr<float>(), rows, r.dim,
            x.stride(0), res ? res->stride(0) : 0, r.tpr, (float)eps);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {y, h, rstd};
}

// (q, scales, h): e4m3 with a scale for each row or each `group` columns.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> rms_norm_fp8(
    torch::Tensor x, torch::Tensor w, c10::optional<torch::Tensor> res,
    double eps, long group) {
  check_matrix(x, x, "x");
  check_weight(w, x);
  const c10::DeviceGuard guard(x.device());
  const long rows = x.size(0), dim = x.size(1);
  if (res) check_matrix(*res, x, "the residual");
  TORCH_CHECK(group == 0 || ((group & (group - 1)) == 0 && group >= 16 &&
                             group <= 256 && dim % group == 0),
              "rms_norm_fp8: groups of 16, 32, 64, 128 or 256 columns that "
              "divide the row, not ", group);
  // a group's columns have neighbouring threads
  const Rows r = plan(rows, dim, group ? group * x.element_size() / 16 : 1);
  auto q = torch::empty({rows, dim},
                        x.options().dtype(at::kFloat8_e4m3fn));
  auto scales = torch::empty({rows, group ? dim / group : 1},
                             x.options().dtype(at::kFloat));
  auto h = torch::empty({res ? rows : 0, dim}, x.options());
  if (rows == 0) return {q, scales, h};
  dispatch(x.scalar_type(), "rms_norm_fp8", [&](auto t) {
    using T = decltype(t);
    rms_fp8_kernel<T>
        <<<dim3(grid_of(r, 4096)), dim3(r.block), 0, stream()>>>(
            (const T*)x.data_ptr(), res ? (const T*)res->data_ptr() : nullptr,
            w.data_ptr(), w.scalar_type() == at::kFloat,
            (unsigned char*)q.data_ptr(), scales.data_ptr<float>(),
            (T*)h.data_ptr(), rows, r.dim, x.stride(0),
            res ? res->stride(0) : 0, r.tpr, (float)eps, (int)group);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {q, scales, h};
}

// (dh, dw): gy and gh are contiguous, x and the residual have contiguous rows.
std::tuple<torch::Tensor, torch::Tensor> rms_norm_bwd(
    torch::Tensor gy, torch::Tensor x, c10::optional<torch::Tensor> res,
    c10::optional<torch::Tensor> gh, torch::Tensor w, torch::Tensor rstd) {
  check_matrix(x, x, "x");
  check_matrix(gy, x, "gy");
  check_weight(w, x);
  const c10::DeviceGuard guard(x.device());
  const long rows = x.size(0), dim = x.size(1);
  TORCH_CHECK(gy.is_contiguous() && rstd.is_cuda() &&
              rstd.device() == x.device() &&
              rstd.scalar_type() == at::kFloat && rstd.numel() == rows &&
              rstd.is_contiguous(),
              "rms_norm_bwd: gy contiguous, rstd float32 for each row");
  if (res) check_matrix(*res, x, "the residual");
  if (gh) {
    check_matrix(*gh, x, "gh");
    TORCH_CHECK(gh->is_contiguous(), "rms_norm_bwd: gh contiguous");
  }
  const Rows r = plan(rows, dim);
  auto dh = torch::empty({rows, dim}, x.options());
  auto dw = torch::empty({dim}, w.options());
  const int grid = grid_of(r, 262144 / r.block);  // four waves on a SIMD
  auto part = torch::empty({grid, dim}, x.options().dtype(at::kFloat));
  if (rows) {
    const int lds = r.block > r.tpr ? r.dim * (int)sizeof(float) : 0;
    dispatch(x.scalar_type(), "rms_norm", [&](auto t) {
      using T = decltype(t);
      rms_bwd_kernel<T><<<dim3(grid), dim3(r.block), lds, stream()>>>(
          (const T*)gy.data_ptr(), (const T*)x.data_ptr(),
          res ? (const T*)res->data_ptr() : nullptr,
          gh ? (const T*)gh->data_ptr() : nullptr, w.data_ptr(),
          w.scalar_type() == at::kFloat, rstd.data_ptr<float>(),
          (T*)dh.data_ptr(), part.data_ptr<float>(), rows, r.dim,
          x.stride(0), res ? res->stride(0) : 0, r.tpr);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  dispatch(w.scalar_type(), "rms_norm", [&](auto t) {
    using W = decltype(t);
    rms_dw_kernel<W><<<dim3((dim + 15) / 16), dim3(256), 0, stream()>>>(
        part.data_ptr<float>(), (W*)dw.data_ptr(), grid, r.dim);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {dh, dw};
}

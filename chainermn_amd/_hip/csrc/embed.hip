// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[t]  = c * W[id_t]                       (zero where id_t is ignored)
//   dW[v] = c * sum of gy[t] over id_t == v   (the whole table, zeros too)
//
// Both are bound by memory.  The gradient is three launches without float
// atomics, so that its sums have one order and two runs agree bit by bit:
//
//   1. embed_sort: counting sort of the tokens by id.  A workgroup owns a
//      range of at most 1024 ids and reads ALL ids (they come from L2): what
//      it counts below its range is its place in the sorted order, so no
//      workgroup waits for another one.
//   2. embed_rows: a wave sums 32 sorted tokens of a slice of columns; rows
//      that begin and end within its tokens are finished, the two at its
//      ends leave partial sums.  So a frequent word costs no more than
//      others.  Rows without a token are zeroed by further waves.
//   3. embed_join: adds up the partial sums of rows that span chunks.

#include "seq_common.h"

namespace {

using namespace seq;

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kMaxBins = 1024;  // ids of a workgroup: 64 KB of counters
constexpr int kChunk = 32;      // sorted tokens of a wave
constexpr int kJoinWaves = 8;

// ids behind this are neither looked up nor summed
template <typename I>
__device__ __forceinline__ long id_at(const I* ids, long t, long vocab,
                                      bool has_ignore, long ignore) {
  const long id = ids[t];
  return (id < 0 || id >= vocab || (has_ignore && id == ignore)) ? -1 : id;
}

template <typename T, int VE, typename I>
__global__ __launch_bounds__(256) void embed_lookup_kernel(
    const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ y,
    long n, long vocab, long dim, long stride, float scale, bool has_ignore,
    long ignore, int lanes) {
  const int rows = 256 / lanes;
  const long t = blockIdx.x * (long)rows + threadIdx.x / lanes;
  if (t >= n) return;
  const long id = ids[t];
  const bool skip = has_ignore && id == ignore;
  const bool bad = id < 0 || id >= vocab;
  const T* src = w + (skip || bad ? 0 : id * stride);
  T* dst = y + t * dim;
  const float none = skip ? 0.f : __builtin_nanf("");
  const long step = (long)lanes * VE;
#pragma unroll 4
  for (long c = (threadIdx.x % lanes) * VE; c < dim; c += step) {
    float r[VE];
    if (skip || bad) {
#pragma unroll
      for (int i = 0; i < VE; ++i) r[i] = none;
    } else {
      load<T, VE>(src + c, r);
#pragma unroll
      for (int i = 0; i < VE; ++i) r[i] *= scale;
    }
    store<T, VE>(dst + c, r);
  }
}

// The lanes of `among` that have this lane's bin.
__device__ __forceinline__ unsigned long long same_bin(
    unsigned long long among, int bin, int bits) {
  for (int b = 0; b < bits; ++b) {
    const bool one = (bin >> b) & 1;
    const unsigned long long m = __ballot(one);
    among &= one ? m : ~m;
  }
  return among;
}

// order[0..m): the tokens by id, those of one id in their own order;
// sorted[0..m): their ids; offsets[v]: the first place of id v, offsets
// [vocab] = m.  Tokens that are ignored or out of range are left out.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(
    const I* __restrict__ ids, long n, long vocab, int range, int bits,
    bool has_ignore, long ignore, int* __restrict__ order,
    int* __restrict__ sorted, int* __restrict__ offsets) {
  extern __shared__ int count[];  // [wave][range]
  __shared__ int below[kSortWaves];
  __shared__ int scan[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long lo = blockIdx.x * (long)range;
  const long hi = lo + range < vocab ? lo + range : vocab;
  const long per = (n + kSortThreads - 1) / kSortThreads * 64;
  const long begin = wave * per;
  const long end = begin + per < n ? begin + per : n;
  int* mine = count + wave * range;
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads)
    count[i] = 0;
  __syncthreads();

  constexpr int U = 8;  // loads in flight
  int less = 0;
  for (long base = begin; base < end; base += 64 * U) {
    long id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long t = base + u * 64 + lane;
      id[u] = t < end ? id_at(ids, t, vocab, has_ignore, ignore) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      less += id[u] >= 0 && id[u] < lo;
      const bool in = id[u] >= lo && id[u] < hi;
      const unsigned long long any = __ballot(in);
      if (any == 0) continue;
      const int bin = in ? int(id[u] - lo) : 0;
      const unsigned long long eq = same_bin(any, bin, bits);
      if (in && lane == __ffsll(eq) - 1) atomicAdd(&mine[bin], __popcll(eq));
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) less += __shfl_xor(less, off, 64);
  if (lane == 0) below[wave] = less;
  __syncthreads();

  // every bin's first place, and every wave's within the bin
  int start = 0;
  for (int i = 0; i < kSortWaves; ++i) start += below[i];
  const int bin0 = threadIdx.x;
  int total = 0;
  if (bin0 < range)
    for (int i = 0; i < kSortWaves; ++i) total += count[i * range + bin0];
  int incl = total;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off, 64);
    if (lane >= off) incl += up;
  }
  if (lane == 63) scan[wave] = incl;
  __syncthreads();
  for (int i = 0; i < wave; ++i) start += scan[i];
  start += incl - total;
  if (bin0 < range) {
    int at = start;
    for (int i = 0; i < kSortWaves; ++i) {
      const int c = count[i * range + bin0];
      count[i * range + bin0] = at;
      at += c;
    }
    if (lo + bin0 < vocab) {
      offsets[lo + bin0] = start;
      if (lo + bin0 == vocab - 1) offsets[vocab] = at;
    }
  }
  __syncthreads();

  for (long base = begin; base < end; base += 64 * U) {
    long id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long t = base + u * 64 + lane;
      id[u] = t < end ? id_at(ids, t, vocab, has_ignore, ignore) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = id[u] >= lo && id[u] < hi;
      const unsigned long long any = __ballot(in);
      if (any == 0) continue;
      const int bin = in ? int(id[u] - lo) : 0;
      const unsigned long long eq = same_bin(any, bin, bits);
      const int leader = in ? __ffsll(eq) - 1 : lane;
      int first = 0;
      if (in && lane == leader) first = atomicAdd(&mine[bin], __popcll(eq));
      first = __shfl(first, leader, 64);
      if (in) {
        const int at = first + __popcll(eq & ((1ull << lane) - 1));
        order[at] = int(base + u * 64 + lane);
        sorted[at] = int(id[u]);
      }
    }
  }
}

// Waves 0 .. chunks * slices - 1: the sums of 32 sorted tokens over a slice
// of 64 * VE columns.  The waves behind them zero the rows without a token.
template <typename T, int VE>
__global__ __launch_bounds__(256) void embed_rows_kernel(
    const T* __restrict__ gy, const int* __restrict__ order,
    const int* __restrict__ sorted, const int* __restrict__ offsets,
    T* __restrict__ dw, float* __restrict__ head, float* __restrict__ tail,
    long vocab, long dim, int chunks, int slices, float scale) {
  const int lane = threadIdx.x & 63;
  long wave = blockIdx.x * 4l + (threadIdx.x >> 6);
  const long sums = (long)chunks * slices;
  if (wave >= sums) {
    const long waves = gridDim.x * 4l - sums;
    float z[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] = 0.f;
    for (long v = wave - sums; v < vocab; v += waves) {
      if (offsets[v] != offsets[v + 1]) continue;
      for (long c = lane * VE; c < dim; c += 64 * VE)
        store<T, VE>(dw + v * dim + c, z);
    }
    return;
  }
  const int chunk = __builtin_amdgcn_readfirstlane(int(wave / slices));
  const long col = (wave % slices) * 64 * VE + lane * VE;
  const int m = offsets[vocab];
  const int p0 = chunk * kChunk;
  if (p0 >= m) return;
  const int len = m - p0 < kChunk ? m - p0 : kChunk;
  const bool on = col < dim;
  const int at = p0 + (lane < len ? lane : 0);
  const int my_tok = order[at], my_id = sorted[at];
  // whether the row goes on in the neighbouring chunks
  const bool before = p0 > 0 && sorted[p0 - 1] == sorted[p0];
  const bool after = p0 + len < m && sorted[p0 + len] == sorted[p0 + len - 1];
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
  bool first = true;  // still in the chunk's first row
  constexpr int U = 8;
  for (int j0 = 0; j0 < len; j0 += U) {
    float g[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tok = __shfl(my_tok, j0 + u < len ? j0 + u : 0, 64);
      if (on && j0 + u < len) {
        load<T, VE>(gy + tok * dim + col, g[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) g[u][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j >= len) break;
      const int id = __builtin_amdgcn_readfirstlane(__shfl(my_id, j, 64));
      const int next = __builtin_amdgcn_readfirstlane(
          __shfl(my_id, j + 1 < len ? j + 1 : j, 64));
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += g[u][i];
      if (j + 1 < len && next == id) continue;
      // the row ends here, or the chunk does
      if (first && before) {
        if (on) store<float, VE>(head + chunk * dim + col, acc);
      } else if (j + 1 == len && after) {
        if (on) store<float, VE>(tail + chunk * dim + col, acc);
      } else if (on) {
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] *= scale;
        store<T, VE>(dw + id * dim + col, acc);
      }
      first = false;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] = 0.f;
    }
  }
}

// A workgroup of a chunk in which a row begins that goes on behind it: its
// tail there and the heads of the chunks up to the row's last token.
template <typename T, int VE>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(
    const int* __restrict__ sorted, const int* __restrict__ offsets,
    const float* __restrict__ head, const float* __restrict__ tail,
    T* __restrict__ dw, long vocab, long dim, float scale) {
  __shared__ float part[kJoinWaves][64 * VE];
  const int chunk = blockIdx.x;
  const int m = offsets[vocab];
  const int p1 = (chunk + 1) * kChunk;
  if (p1 >= m) return;
  const int id = sorted[p1];
  if (sorted[p1 - 1] != id || offsets[id] < chunk * kChunk) return;
  const int last = (offsets[id + 1] - 1) / kChunk;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long col = blockIdx.y * 64l * VE + lane * VE;
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
  if (col < dim) {
    if (wave == 0) load<float, VE>(tail + chunk * dim + col, acc);
#pragma unroll 8
    for (int c = chunk + 1 + wave; c <= last; c += kJoinWaves) {
      float r[VE];
      load<float, VE>(head + c * dim + col, r);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += r[i];
    }
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) part[wave][lane * VE + i] = acc[i];
  __syncthreads();
  if (wave != 0 || col >= dim) return;
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] += part[w][lane * VE + i];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] *= scale;
  store<T, VE>(dw + id * dim + col, acc);
}

void check_ids(const torch::Tensor& ids, const char* what) {
  TORCH_CHECK(ids.is_cuda() && ids.is_contiguous() &&
              (ids.scalar_type() == at::kLong ||
               ids.scalar_type() == at::kInt),
              what, ": ids must be a contiguous int32 or int64 GPU tensor");
}

}  // namespace

torch::Tensor embed_lookup(torch::Tensor ids, torch::Tensor w, double scale,
                           bool has_ignore, long ignore) {
  check_ids(ids, "embed_lookup");
  TORCH_CHECK(w.is_cuda() && w.dim() == 2 && w.device() == ids.device() &&
              w.size(0) > 0 && w.size(1) > 0 &&
              (w.stride(1) == 1 || w.size(1) == 1),
              "embed_lookup: the table must be a non-empty matrix of "
              "contiguous rows on the ids' GPU");
  const c10::DeviceGuard guard(w.device());
  const long n = ids.numel(), dim = w.size(1);
  auto shape = ids.sizes().vec();
  shape.push_back(dim);
  auto y = torch::empty(shape, w.options());
  if (n == 0) return y;
  int ve = vector_width(w.data_ptr(), dim, w.stride(0), w.element_size());
  const long nvec = dim / ve;
  int lanes = 64;  // of a row; a wave takes several short ones
  while (lanes > 1 && lanes / 2 >= nvec) lanes /= 2;
  const long blocks = (n + 256 / lanes - 1) / (256 / lanes);
  TORCH_CHECK(blocks < (1l << 31), "embed_lookup: too many tokens");
  dispatch_vec(w.scalar_type(), ve, "embed_lookup", [&](auto t, auto width) {
    using T = decltype(t);
    constexpr int VE = decltype(width)::value;
    auto go = [&](auto i) {
      using I = decltype(i);
      embed_lookup_kernel<T, VE, I><<<dim3(blocks), dim3(256), 0, stream()>>>(
          (const I*)ids.data_ptr(), (const T*)w.data_ptr(),
          (T*)y.data_ptr(), n, w.size(0), dim, w.stride(0), (float)scale,
          has_ignore, ignore, lanes);
    };
    if (ids.scalar_type() == at::kLong) go(long());
    else go(int());
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return y;
}

torch::Tensor embed_grad(torch::Tensor ids, torch::Tensor gy, long vocab,
                         double scale, bool has_ignore, long ignore) {
  check_ids(ids, "embed_grad");
  const long n = ids.numel();
  TORCH_CHECK(gy.is_cuda() && gy.device() == ids.device() &&
              gy.dim() >= 1 && gy.is_contiguous() && gy.size(-1) > 0 &&
              gy.numel() == n * gy.size(-1) && vocab > 0,
              "embed_grad: gy must be contiguous, one row for each id");
  // places and ids are held in 32 bits
  TORCH_CHECK(n < (1l << 31) - 64 * kSortThreads && vocab < (1l << 31) - 1,
              "embed_grad: fewer than 2^31 tokens and rows");
  const c10::DeviceGuard guard(gy.device());
  const long dim = gy.size(-1);
  auto dw = torch::empty({vocab, dim}, gy.options());
  const auto ints = gy.options().dtype(at::kInt);
  // a range for each of 256 workgroups, or as many as 1024 ids each take
  int range = int((vocab + 255) / 256);
  if (range > kMaxBins) range = kMaxBins;
  int bits = 0;
  while ((1 << bits) < range) ++bits;
  const int groups = int((vocab + range - 1) / range);
  auto places = torch::empty({2 * n + vocab + 1}, ints);
  int* order = places.data_ptr<int>();
  int* sorted = order + n;
  int* offsets = sorted + n;
  const int lds = kSortWaves * range * (int)sizeof(int);
  auto sort = [&](auto i) {
    using I = decltype(i);
    embed_sort_kernel<I><<<dim3(groups), dim3(kSortThreads), lds, stream()>>>(
        (const I*)ids.data_ptr(), n, vocab, range, bits, has_ignore, ignore,
        order, sorted, offsets);
  };
  if (ids.scalar_type() == at::kLong) sort(long());
  else sort(int());
  C10_HIP_KERNEL_LAUNCH_CHECK();

  const int ve = vector_width(gy.data_ptr(), dim, dim, gy.element_size());
  const int chunks = int((n + kChunk - 1) / kChunk);
  auto parts = torch::empty({2, chunks, dim},
                            gy.options().dtype(at::kFloat));
  float* head = parts.data_ptr<float>();
  float* tail = head + (long)chunks * dim;
  const int slices = int((dim + 64 * ve - 1) / (64 * ve));
  const long zero_waves = vocab < 4096 ? vocab : 4096;
  const long blocks = ((long)chunks * slices + zero_waves + 3) / 4;
  TORCH_CHECK(blocks < (1l << 31) && slices < 65536,
              "embed_grad: too many elements");
  dispatch_vec(gy.scalar_type(), ve, "embed_grad", [&](auto t, auto width) {
    using T = decltype(t);
    constexpr int VE = decltype(width)::value;
    embed_rows_kernel<T, VE><<<dim3(blocks), dim3(256), 0, stream()>>>(
        (const T*)gy.data_ptr(), order, sorted, offsets, (T*)dw.data_ptr(),
        head, tail, vocab, dim, chunks, slices, (float)scale);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    if (chunks > 1)
      embed_join_kernel<T, VE>
          <<<dim3(chunks, slices), dim3(64 * kJoinWaves), 0, stream()>>>(
              sorted, offsets, head, tail, (T*)dw.data_ptr(), vocab, dim,
              (float)scale);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dw;
}

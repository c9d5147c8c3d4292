// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[t]  = c * W[id_t]                       (zero where id_t is ignored)
//   dW[v] = c * sum of gy[t] over id_t == v   (the whole table, zeros too)
//
// 32768 tokens of 32000 x 1024 in fp32, 8791 rows of them: the lookup takes 38
// us, 4.5 TB/s of what it has to move, and the gradient 81 us: 55 us for
// embed_rows, 4.8 TB/s, which memory bounds, 18 us for the order and 7 us for
// embed_join, which latency does, with memory idle.
// (With one sorting pass, in which every workgroup reads all ids, the order
// alone took 50 us.)
//
// The gradient has no float atomics, so its sums have one order and two runs
// agree bit by bit:
//
//   1. embed_split and embed_sort: a stable counting sort of the tokens by
//      id, first 1024 tokens of a workgroup by the low bits of their ids,
//      then each of these buckets by the others.  A bucket's workgroup finds
//      its place in the order from the counts of all of them, so none waits
//      for another one.  Low bits, because the frequent words of a vocabulary
//      sorted by frequency are neighbours.  16 waves: the bucket of the most
//      frequent word lasts longest.  (262144 tokens, 7% of them one word, both
//      passes: 402 us; with 8 waves 429 us.)  A bucket's
//      workgroup sorts a frequent word alone: where half of 32768 tokens are
//      one word, the gradient takes 112 us instead of 64 us (the same input
//      again and again, in the caches), so padding should be ignored.
//   2. embed_rows: a wave sums 8 to 32 sorted tokens of some columns; rows
//      that begin and end within its tokens are finished, the two at its
//      ends leave partial sums.  So a frequent word costs no more than
//      others here.  Rows without a token are zeroed by further waves.
//   3. embed_join: adds up the partial sums of rows that span chunks.

#include "seq_common.h"

namespace {

using namespace seq;

constexpr int kSplitThreads = 1024, kSplitWaves = kSplitThreads / 64;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxBins = 512;     // ids of a workgroup of embed_sort
constexpr int kMaxPieces = 1024;  // workgroups of embed_split
constexpr int kJoinWaves = 8;

// The column at which a lane reads and writes: the last vector of a row of
// odd length is moved back onto the one before it, and both lanes compute the
// same.  Rows shorter than a vector are read by elements.
template <int VE>
__device__ __forceinline__ long column(long c, long dim) {
  return c + VE <= dim ? c : dim < VE ? 0 : dim - VE;
}

// ids behind this are neither looked up nor summed
template <typename I>
__device__ __forceinline__ long id_at(const I* ids, long t, long vocab,
                                      bool has_ignore, long ignore) {
  const long id = ids[t];
  return (id < 0 || id >= vocab || (has_ignore && id == ignore)) ? -1 : id;
}

template <typename T, typename I>
__global__ __launch_bounds__(256) void embed_lookup_kernel(
    const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ y,
    long n, long vocab, long dim, long stride, float scale, bool has_ignore,
    long ignore, int lanes) {
  constexpr int VE = kWidth<T>;
  const int rows = 256 / lanes;
  const long t = blockIdx.x * (long)rows + threadIdx.x / lanes;
  if (t >= n) return;
  const long id = ids[t];
  const bool skip = has_ignore && id == ignore;
  const bool bad = id < 0 || id >= vocab;
  const T* src = w + id * stride;
  T* dst = y + t * dim;
  const long step = (long)lanes * VE;
  if (skip || bad) {
    float r[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) r[i] = skip ? 0.f : __builtin_nanf("");
    for (long c = (threadIdx.x % lanes) * VE; c < dim; c += step)
      store<T, VE, true>(dst + column<VE>(c, dim), r, dim);
    return;
  }
  constexpr int U = 4;  // vectors in flight
  for (long c0 = (threadIdx.x % lanes) * VE; c0 < dim; c0 += U * step) {
    float r[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load<T, VE>(src + column<VE>(c0 + u * step, dim), r[u], dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u * step >= dim) break;
#pragma unroll
      for (int i = 0; i < VE; ++i) r[u][i] *= scale;
      store<T, VE, true>(dst + column<VE>(c0 + u * step, dim), r[u], dim);
    }
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

// The exclusive sum over a workgroup of WAVES waves, and the whole sum.
template <int WAVES>
__device__ __forceinline__ int scan(int v, int* lds, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off, 64);
    if (lane >= off) incl += up;
  }
  if (lane == 63) lds[wave] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i < wave) before += lds[i];
    total += lds[i];
  }
  __syncthreads();
  *all = total;
  return before + incl - v;
}

// A stable counting sort of `n` items by a workgroup: fetch(p) is item p (an
// id and a token, or a negative id), bin(item) its bin or -1 for none, and
// emit(item, place) gets its place.  count is [WAVES][bins], and begin(bin,
// first, n) gets each bin's first place and size.  Each wave takes a run of
// the items, four of each lane's at once.
template <int WAVES, typename F, typename B, typename G, typename E>
__device__ __forceinline__ void counting_sort(long n, int bins, int bits,
                                              int* count, int* lds, F fetch,
                                              B bin, G begin, E emit) {
  constexpr int U = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long per = (n + 64 * WAVES - 1) / (64 * WAVES) * 64;
  const long first = wave * per, last = first + per < n ? first + per : n;
  int* mine = count + wave * bins;
  for (int i = threadIdx.x; i < WAVES * bins; i += 64 * WAVES) count[i] = 0;
  __syncthreads();
  for (long p0 = first; p0 < last; p0 += 64 * U) {
    int2 it[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long p = p0 + u * 64 + lane;
      it[u] = p < last ? fetch(p) : make_int2(-1, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = it[u].x >= 0 ? bin(it[u]) : -1;
      const unsigned long long any = __ballot(b >= 0);
      if (any == 0) continue;
      const unsigned long long eq = same_bin(any, b, bits);
      if (b >= 0 && lane == __ffsll(eq) - 1)
        atomicAdd(&mine[b], __popcll(eq));
    }
  }
  __syncthreads();
  int before = 0;  // of the bins of earlier rounds
  for (int b0 = 0; b0 < bins; b0 += 64 * WAVES) {
    const int b = b0 + threadIdx.x;
    int total = 0, all;
    if (b < bins)
      for (int i = 0; i < WAVES; ++i) total += count[i * bins + b];
    int at = before + scan<WAVES>(total, lds, &all);
    before += all;
    if (b < bins) {
      begin(b, at, total);
      for (int i = 0; i < WAVES; ++i) {
        const int c = count[i * bins + b];
        count[i * bins + b] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  for (long p0 = first; p0 < last; p0 += 64 * U) {
    int2 it[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long p = p0 + u * 64 + lane;
      it[u] = p < last ? fetch(p) : make_int2(-1, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = it[u].x >= 0 ? bin(it[u]) : -1;
      const unsigned long long any = __ballot(b >= 0);
      if (any == 0) continue;
      const unsigned long long eq = same_bin(any, b, bits);
      const int leader = b >= 0 ? __ffsll(eq) - 1 : lane;
      int at = 0;
      if (b >= 0 && lane == leader) at = atomicAdd(&mine[b], __popcll(eq));
      at = __shfl(at, leader, 64) + __popcll(eq & ((1ull << lane) - 1));
      if (b >= 0) emit(it[u], at);
    }
  }
}

// A piece of the tokens, sorted by bucket: piece[0..) are (id, token), and
// starts[bucket][workgroup] each bucket's first place, up to one behind the
// last bucket.  Tokens that are ignored or out of range are left out.
template <typename I>
__global__ __launch_bounds__(kSplitThreads) void embed_split_kernel(
    const I* __restrict__ ids, long n, long vocab, long per, int bucket_bits,
    bool has_ignore, long ignore, int2* __restrict__ pieces,
    int* __restrict__ starts) {
  extern __shared__ int count[];  // [wave][buckets]
  __shared__ int lds[kSplitWaves];
  const long p0 = blockIdx.x * per;
  const long here = p0 + per < n ? per : n - p0;
  const int buckets = 1 << bucket_bits;
  counting_sort<kSplitWaves>(
      here, buckets, bucket_bits, count, lds,
      [&](long p) {
        return make_int2(
            int(id_at(ids, p0 + p, vocab, has_ignore, ignore)), int(p0 + p));
      },
      [&](int2 it) { return it.x & (buckets - 1); },
      [&](int b, int at, int size) {
        starts[(long)b * gridDim.x + blockIdx.x] = at;
        if (b == buckets - 1)
          starts[(long)buckets * gridDim.x + blockIdx.x] = at + size;
      },
      [&](int2 it, int at) { pieces[p0 + at] = it; });
}

// A bucket of all pieces, or `bins` of its ids, sorted by id.  order[0..m):
// the tokens, those of one id in their own order; sorted[0..m): their ids;
// range[v]: the places of id v; *tokens = m.
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(
    const int2* __restrict__ pieces, const int* __restrict__ starts, int n,
    long per, long vocab, int bucket_bits, int bins, int bits, int parts,
    int* __restrict__ order, int* __restrict__ sorted,
    int2* __restrict__ range, int* __restrict__ tokens) {
  extern __shared__ int count[];  // [wave][bins]
  __shared__ int piece[kMaxPieces + 1];  // first item of a piece in the list
  __shared__ int from[kMaxPieces];       // and its place in the pieces
  __shared__ int lds[kSortWaves];
  __shared__ int below;
  const int bucket = blockIdx.x / parts, part = blockIdx.x % parts;
  const int* a = starts + (long)bucket * n;
  int items = 0, place = 0, all;
  for (int g0 = 0; g0 < n; g0 += kSortThreads) {
    const int g = g0 + threadIdx.x;
    const int at = g < n ? a[g] : 0, size = g < n ? a[n + g] - at : 0;
    const int first = scan<kSortWaves>(size, lds, &all);
    if (g < n) {
      piece[g] = items + first;
      from[g] = int(g * per) + at;
    }
    items += all;
    scan<kSortWaves>(at, lds, &all);
    place += all;
  }
  if (threadIdx.x == 0) {
    piece[n] = items;
    below = 0;
  }
  if (blockIdx.x == 0) {
    int m = 0;
    for (int g = threadIdx.x; g < n; g += kSortThreads)
      m += starts[((long)n << bucket_bits) + g];
    scan<kSortWaves>(m, lds, &all);
    if (threadIdx.x == 0) *tokens = all;
  }
  __syncthreads();
  auto item = [&](long p) {
    int lo = 0, hi = n - 1;  // the last piece that begins at or before p
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (piece[mid] <= p) lo = mid;
      else hi = mid - 1;
    }
    return pieces[from[lo] + (int(p) - piece[lo])];
  };
  const int bin0 = part * bins;
  if (part > 0) {  // what the bucket's parts before this one hold
    int less = 0;
    for (int p = threadIdx.x; p < items; p += kSortThreads)
      less += (item(p).x >> bucket_bits) < bin0;
    atomicAdd(&below, less);
    __syncthreads();
    place += below;
  }
  counting_sort<kSortWaves>(
      items, bins, bits, count, lds, item,
      [&](int2 it) {
        const int b = (it.x >> bucket_bits) - bin0;
        return b >= 0 && b < bins ? b : -1;
      },
      [&](int b, int at, int size) {
        const long id = ((long)(bin0 + b) << bucket_bits) + bucket;
        if (id < vocab)
          range[id] = make_int2(place + at, place + at + size);
      },
      [&](int2 it, int at) {
        order[place + at] = it.y;
        sorted[place + at] = it.x;
      });
}

// Waves 0 .. chunks * slices - 1: the sums of `size` sorted tokens over a
// slice of 64 * VE columns.  The waves behind them zero the rows without a
// token.
template <typename T>
__global__ __launch_bounds__(256) void embed_rows_kernel(
    const T* __restrict__ gy, const int* __restrict__ order,
    const int* __restrict__ sorted, const int2* __restrict__ range,
    const int* __restrict__ tokens, T* __restrict__ dw,
    float* __restrict__ head, float* __restrict__ tail,
    long vocab, long dim, int size, int chunks, int slices, float scale) {
  constexpr int VE = kWidth<T>;
  const int lane = threadIdx.x & 63;
  long wave = blockIdx.x * 4l + (threadIdx.x >> 6);
  const long sums = (long)chunks * slices;
  if (wave >= sums) {
    const long waves = gridDim.x * 4l - sums;
    float z[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] = 0.f;
    for (long v = wave - sums; v < vocab; v += waves) {
      const int2 r = range[v];
      if (r.x != r.y) continue;
      for (long c = lane * VE; c < dim; c += 64 * VE)
        store<T, VE, true>(dw + v * dim + column<VE>(c, dim), z, dim);
    }
    return;
  }
  const int chunk = __builtin_amdgcn_readfirstlane(int(wave / slices));
  long col = (wave % slices) * 64 * VE + lane * VE;
  const bool on = col < dim;
  col = column<VE>(col, dim);
  const int m = *tokens;
  const int p0 = chunk * size;
  if (p0 >= m) return;
  const int len = m - p0 < size ? m - p0 : size;
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
      load<T, VE>(gy + tok * dim + col, g[u], dim);
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
        if (on) store<float, VE>(head + chunk * dim + col, acc, dim);
      } else if (j + 1 == len && after) {
        if (on) store<float, VE>(tail + chunk * dim + col, acc, dim);
      } else if (on) {
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] *= scale;
        store<T, VE, true>(dw + id * dim + col, acc, dim);
      }
      first = false;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] = 0.f;
    }
  }
}

// A row that begins in a chunk and goes on behind it: its tail there and the
// heads of the chunks up to its last token.  A wave has a chunk; rows of more
// than 16 parts are then summed by all eight waves.
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(
    const int* __restrict__ sorted, const int2* __restrict__ range,
    const int* __restrict__ tokens, const float* __restrict__ head,
    const float* __restrict__ tail, T* __restrict__ dw, long dim, int size,
    float scale) {
  constexpr int VE = kWidth<T>;
  __shared__ float part[kJoinWaves][64 * VE];
  __shared__ int3 rows[kJoinWaves];  // of many parts: id, first, last chunk
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long col = blockIdx.y * 64l * VE + lane * VE;
  const bool on = col < dim;
  col = column<VE>(col, dim);
  const int m = *tokens;

  // the parts of a row that are `step` chunks apart
  auto sum = [&](int chunk, int from, int last, int step, float (&acc)[VE]) {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.f;
    if (!on) return;
    if (from == chunk + 1)
      load<float, VE>(tail + chunk * dim + col, acc, dim);
#pragma unroll 8
    for (int c = from; c <= last; c += step) {
      float r[VE];
      load<float, VE>(head + c * dim + col, r, dim);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += r[i];
    }
  };
  auto finish = [&](int id, float (&acc)[VE]) {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] *= scale;
    store<T, VE, true>(dw + id * dim + col, acc, dim);
  };

  const int chunk = blockIdx.x * kJoinWaves + wave;
  const long p1 = (chunk + 1l) * size;
  int3 row = make_int3(-1, 0, 0);
  if (p1 < m && sorted[p1 - 1] == sorted[p1]) {
    const int id = sorted[p1];
    const int2 r = range[id];
    if (r.x >= p1 - size) row = make_int3(id, chunk, (r.y - 1) / size);
  }
  const bool many = row.z - row.y > 16;
  if (lane == 0) rows[wave] = many ? row : make_int3(-1, 0, 0);
  if (row.x >= 0 && !many) {
    float acc[VE];
    sum(row.y, row.y + 1, row.z, 1, acc);
    finish(row.x, acc);
  }
  __syncthreads();
  for (int k = 0; k < kJoinWaves; ++k) {
    const int3 r = rows[k];
    if (r.x < 0) continue;  // for all waves alike
    float acc[VE];
    sum(r.y, r.y + 1 + wave, r.z, kJoinWaves, acc);
#pragma unroll
    for (int i = 0; i < VE; ++i) part[wave][lane * VE + i] = acc[i];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] += part[w][lane * VE + i];
      finish(r.x, acc);
    }
    __syncthreads();
  }
}

// The whole gradient of a few tokens and rows in one launch: a workgroup looks
// for its row among all ids, each wave in a run of them.
// grid: (vocab, slices).
template <typename T, typename I>
__global__ __launch_bounds__(kSplitThreads) void embed_direct_kernel(
    const I* __restrict__ ids, const T* __restrict__ gy, T* __restrict__ dw,
    long n, long dim, bool has_ignore, long ignore, float scale) {
  constexpr int VE = kWidth<T>;
  __shared__ float part[kSplitWaves][64 * VE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x, col0 = blockIdx.y * 64l * VE;
  const long col = column<VE>(col0 + lane * VE, dim);
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
  const long per = (n + kSplitThreads - 1) / kSplitThreads * 64;
  const long first = wave * per, last = first + per < n ? first + per : n;
  if (!(has_ignore && row == ignore)) {
    for (long p0 = first; p0 < last; p0 += 64) {
      const bool is = p0 + lane < last && ids[p0 + lane] == row;
      unsigned long long left = __ballot(is);
      while (left) {
        constexpr int U = 4;  // rows in flight
        float g[U][VE];
        int found = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = __ffsll(left) - 1;
          if (at >= 0) {
            load<T, VE>(gy + (p0 + at) * dim + col, g[u], dim);
            left &= left - 1;
            ++found;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < found)
#pragma unroll
            for (int i = 0; i < VE; ++i) acc[i] += g[u][i];
      }
    }
  }
  // a row's odd end is moved onto the vector before it, here too
#pragma unroll
  for (int i = 0; i < VE; ++i)
    if (col - col0 + i >= lane * VE) part[wave][col - col0 + i] = acc[i];
  __syncthreads();
  for (int c = threadIdx.x; c < 64 * VE && col0 + c < dim;
       c += kSplitThreads) {
    float sum = 0.f;
    for (int w = 0; w < kSplitWaves; ++w) sum += part[w][c];
    dw[row * dim + col0 + c] = T(sum * scale);
  }
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
  const int ve = 16 / (int)w.element_size();
  const long nvec = (dim + ve - 1) / ve;
  int lanes = 64;  // of a row; a wave takes several short ones
  while (lanes > 1 && lanes / 2 >= nvec) lanes /= 2;
  const long blocks = (n + 256 / lanes - 1) / (256 / lanes);
  check_grid(blocks, 256, "embed_lookup");
  auto shape = ids.sizes().vec();
  shape.push_back(dim);
  auto y = torch::empty(shape, w.options());
  if (n == 0) return y;
  dispatch(w.scalar_type(), "embed_lookup", [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto i) {
      using I = decltype(i);
      embed_lookup_kernel<T, I><<<dim3(blocks), dim3(256), 0, stream()>>>(
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
  TORCH_CHECK(n < (1l << 30) && vocab < (1l << 30),
              "embed_grad: fewer than 2^30 tokens and rows");
  const c10::DeviceGuard guard(gy.device());
  const long dim = gy.size(-1);
  auto dw = torch::empty({vocab, dim}, gy.options());
  const int ve = 16 / (int)gy.element_size();
  const int slices = int((dim + 64 * ve - 1) / (64 * ve));
  // A row of the table for each workgroup, while they are two rounds of this
  // GPU at most and there are no more tokens than a wave finds quickly.  (1280
  // tokens: 512 rows of 256 in fp32 5 us, by the sort 22 us; 256 rows of 1024 6
  // us, 21 us.  4096 tokens, 1024 rows of 256: 7 us, 23 us, and 4096 rows 17
  // us, 23 us; 16 rows of 1024 15 us, 24 us.  Only one word is the worst, since
  // its row's workgroup sums all of it: 4096 tokens 45 us.)
  if (vocab * slices <= 1024 && n <= 4096) {
    dispatch(gy.scalar_type(), "embed_grad", [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto i) {
        using I = decltype(i);
        embed_direct_kernel<T, I>
            <<<dim3(vocab, slices), dim3(kSplitThreads), 0, stream()>>>(
                (const I*)ids.data_ptr(), (const T*)gy.data_ptr(),
                (T*)dw.data_ptr(), n, dim, has_ignore, ignore, (float)scale);
      };
      if (ids.scalar_type() == at::kLong) go(long());
      else go(int());
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return dw;
  }
  // 256 buckets, or 512 where these have 512 ids and more; above 2^18 ids a
  // bucket is sorted in parts
  int bucket_bits = 0;
  while (bucket_bits < 8 && (1l << bucket_bits) < vocab) ++bucket_bits;
  while (bucket_bits < 9 && (vocab >> bucket_bits) >= kMaxBins) ++bucket_bits;
  const int buckets = 1 << bucket_bits;
  const long of_bucket = (vocab + buckets - 1) / buckets;
  const int bins = int(of_bucket < kMaxBins ? of_bucket : kMaxBins);
  const int parts = int((of_bucket + bins - 1) / bins);
  int bits = 0;
  while ((1 << bits) < bins) ++bits;
  // pieces of 1024 tokens, or as many as make 1024 pieces
  const long per = std::max((long)kSplitThreads,
                            (n + kMaxPieces * 64l - 1) / (kMaxPieces * 64l) *
                                64);
  const int pieces = int((n + per - 1) / per);
  const long starts = (buckets + 1l) * pieces;
  auto space = torch::empty({4 * n + 2 * vocab + starts + 1},
                            gy.options().dtype(at::kInt));
  int2* range = reinterpret_cast<int2*>(space.data_ptr<int>());
  int2* piece = range + vocab;
  int* order = reinterpret_cast<int*>(piece + n);
  int* sorted = order + n;
  int* start = sorted + n;
  int* tokens = start + starts;
  if (n) {
    const int lds = kSplitWaves * buckets * (int)sizeof(int);
    auto split = [&](auto i) {
      using I = decltype(i);
      embed_split_kernel<I>
          <<<dim3(pieces), dim3(kSplitThreads), lds, stream()>>>(
              (const I*)ids.data_ptr(), n, vocab, per, bucket_bits,
              has_ignore, ignore, piece, start);
    };
    if (ids.scalar_type() == at::kLong) split(long());
    else split(int());
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  embed_sort_kernel<<<dim3(buckets * parts), dim3(kSortThreads),
                      kSortWaves * bins * (int)sizeof(int), stream()>>>(
      piece, start, pieces, per, vocab, bucket_bits, bins, bits, parts,
      order, sorted, range, tokens);
  C10_HIP_KERNEL_LAUNCH_CHECK();

  // sorted tokens of a wave: 32, or fewer until four waves have work on each
  // SIMD (22500 rows of 1520 bytes at 16: 32 us, at 32: 35 us)
  int size = 32;
  while (size > 8 && (n + size - 1) / size * slices < 4096) size /= 2;
  const int chunks = int((n + size - 1) / size);
  auto sums = torch::empty({2, chunks, dim},
                            gy.options().dtype(at::kFloat));
  float* head = sums.data_ptr<float>();
  float* tail = head + (long)chunks * dim;
  const long zero_waves = vocab < 4096 ? vocab : 4096;
  const long blocks = ((long)chunks * slices + zero_waves + 3) / 4;
  check_grid(blocks, 256, "embed_grad");
  TORCH_CHECK(slices < 65536, "embed_grad: rows of too many elements");
  dispatch(gy.scalar_type(), "embed_grad", [&](auto t) {
    using T = decltype(t);
    embed_rows_kernel<T><<<dim3(blocks), dim3(256), 0, stream()>>>(
        (const T*)gy.data_ptr(), order, sorted, range, tokens,
        (T*)dw.data_ptr(), head, tail, vocab, dim, size, chunks, slices,
        (float)scale);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    if (chunks > 1)
      embed_join_kernel<T>
          <<<dim3((chunks + kJoinWaves - 1) / kJoinWaves, slices),
             dim3(64 * kJoinWaves), 0, stream()>>>(
              sorted, range, tokens, head, tail, (T*)dw.data_ptr(), dim,
              size, (float)scale);
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dw;
}

// Linear attention with a decay for each head.
//
//   S_t = lam S_(t-1) + k_t^T v_t,   o_t = c q_t S_t,   lam = exp(log_decay)
//
// with a state S of dk x dv for each sequence and head, held in fp32.
//
// Chunked form.  Over a chunk of n tokens (i, j = 0 .. n-1) with the state S
// before it:
//
//   o_i = c (lam^(i+1) q_i S + sum_(j<=i) lam^(i-j) (q_i . k_j) v_j)
//   S  <- lam^n S + sum_j lam^(n-1-j) k_j^T v_j
//
// Backward.  With G_t = dL/dS_t = c q_t^T do_t + lam G_(t+1):
//
//   dq_t = c do_t S_t^T,   dv_t = k_t G_t,   dk_t = v_t G_t^T,   dS_0 = lam G_1
//
// so each gradient is the same form again, with other tensors in the places
// of q, k and v: dq runs forwards in time over (do, v, k), dv backwards over
// (k, q, do) and dk backwards over (v, do, q).  One kernel computes all four;
// a call's problems are "roles" of one launch.  Backwards in time a token
// sees the carry with lam^(n-1-i), and the carry takes lam^(j+1).
//
// Chunks of 32 tokens: the operands of the next product over tokens.  Chunks
// of 64 halve the work on the state for each token, but take the registers of
// the second workgroup of a CU (2 x 16384 tokens, 8 heads of 128, trained, in
// bf16: 381 us with 32, 443 us with 64).  A wave has 16 columns of the state;
// with 32 the same took 388 us instead of 348 us.
//
// What bounds it: forward the memory, where there are many heads of 64 (512 x
// 64 tokens, 16 heads, fp32: 144 us, 4.7 TB/s of what it has to move; with half
// of the tokens there 111 us, 4.3 TB/s).  Otherwise the instructions of a
// chunk, whose phases lie between three barriers: backward of the same 310 us
// and 257 us, 3.0 and 2.6 TB/s, vector pipes 52% and LDS 40% busy; 128 x 512
// tokens, 4 heads of 128 in bf16, 75 us and 187 us.  2 x 16384 tokens, 8 heads
// of 128: forward 117 us, of which states of segments and joining them 40 us;
// backward 241 us.  (Pairs of figures for a choice were taken side by side,
// with the rest as it was then, and may differ from these.)
//
// Long sequences and few heads: the length is cut into segments.  The states
// of the segments alone come first, a scan joins them, and the same kernel
// then starts every segment from its own state.
//
// All products run on bf16 matrix instructions (16x16x32) with fp32 sums:
// a value is cut into terms of 8 bits of mantissa each, exactly: bf16 is one
// term, fp16 two, fp32 three.  They are cut off, not rounded, so the second
// is below 2^-7 of the first one's power of two and the third below 2^-15.  Of
// a product of three terms each, those of second with third and of third with
// third terms are left out, less than 2^-21 of it.  A result that is itself
// rounded to 16 bits, by up to 2^-11 (fp16) or 2^-8 (bf16), takes scores and
// states with two terms (2^-15), and leaves out second with second terms
// (2^-14, fp16 only).  What is left out has the sign of the product.  A term
// below 2^-126 counts as zero, so that fp32 values below 2^-110 have fewer bits.
// The state is fp32 throughout, and what is added to it is a product of three
// terms.
//
// The contraction index of a matrix instruction may be permuted if both
// operands are, so that the accumulators of the state and the scores (four
// consecutive rows for a lane) are operands of the next product as they
// stand: lane group g holds 4g..4g+3 and 16+4g..16+4g+3 of 32.

#include "seq_common.h"

namespace {

using namespace seq;

using frag = vec<bf16, 8>;
using acc4 = vec<float, 4>;
using half4 = vec<short, 4>;

constexpr int kThreads = 256;  // of the kernels other than chunk_kernel
constexpr int kChunk = 32;  // tokens
constexpr float kLog2e = 1.44269504088896340736f;

struct Operand {
  const void* p;
  long b, t, h;  // strides in elements; the last one is 1
};

struct Role {
  Operand q, k, v;
  void* out;           // [batch, length, heads, dv]
  const float* first;  // state that comes in, or null
  float* last;         // state that goes out, or null
  int dk, dv;          // of this role
  float* states;       // [batch * heads][segments][D * D], in lane order
  bool turned;         // states and ends are of the transposed state
  bool reverse;
  float intra, inter, gain;  // factors of scores, q S, and k^T v
};

struct Problem {
  Role role[3];
  const float* log_decay;
  const void* lengths;  // or null
  bool long_lengths;
  int batch, length, heads, roles;
  int segments, per_segment;  // tokens of a segment, a multiple of a chunk
};

__device__ __forceinline__ long length_of(const Problem& pr, int b) {
  if (!pr.lengths) return pr.length;
  const long n = pr.long_lengths ? ((const long*)pr.lengths)[b]
                                 : ((const int*)pr.lengths)[b];
  return n < 0 ? 0 : n < pr.length ? n : pr.length;
}

// exp(-200) is zero in fp32, and 0 * log_decay has to be 0; NaN stays
__device__ __forceinline__ float decay_of(const Problem& pr, int h) {
  const float ld = pr.log_decay[h];
  return ld < -200.f ? -200.f : ld;
}

// A buffer resource of `bytes`: reads behind it give zero, writes are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p,
                                                         int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes,
                                           0x00027000);
}
constexpr int kBehind = 0x7ffffff0;  // an offset behind any of them

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
template <>
constexpr int kTerms<fp16> = 2;

// Terms are cut off, not rounded: each is exact in bf16, and three of them
// are the whole of an fp32.  A term is the upper half of its word.
template <int N>
__device__ __forceinline__ void cut(float x, unsigned (&term)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    term[i] = __float_as_uint(x);
    if (i + 1 < N) x -= __uint_as_float(term[i] & 0xffff0000u);
  }
}

// The upper halves of two words, a below b.
__device__ __forceinline__ unsigned pair(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302);
}

// Tiles of bf16 in LDS are row-major with a padded pitch, so that every
// fragment's address is a lane's base and a constant.  The pads put the eight
// rows that are read at once on all banks: 32 bytes where a row gives 32 of
// them (the transposing reads), 16 bytes where it gives 16.
//
// A tile whose rows are only read as fragments keeps its columns in the order
// of the lanes: of 32 columns, 4g..4g+3 and 16+4g..16+4g+3 are neighbours.
__device__ __forceinline__ int in_lane_order(int col) {
  return (col & ~31) | ((col & 12) << 1) | ((col & 16) >> 2) | (col & 3);
}

// Fragment of 16 rows from `row`, 32 columns from `col`, of a tile in lane
// order.
template <int PITCH>
__device__ __forceinline__ frag by_row(const short* tile, int row, int col,
                                       int lane) {
  return *reinterpret_cast<const frag*>(tile + (row + (lane & 15)) * PITCH +
                                        col + (lane >> 4) * 8);
}

// The same of a tile in its own order.
template <int PITCH>
__device__ __forceinline__ frag by_row_plain(const short* tile, int row,
                                             int col, int lane) {
  const short* p = tile + (row + (lane & 15)) * PITCH + col + (lane >> 4) * 4;
  union {
    half4 h[2];
    frag f;
  } u;
  u.h[0] = *reinterpret_cast<const half4*>(p);
  u.h[1] = *reinterpret_cast<const half4*>(p + 16);
  return u.f;
}

// Fragment of 16 columns from `col`, 32 rows from `row`: the transposing
// read gives a lane four rows of one column.
template <int PITCH>
__device__ __forceinline__ frag by_col(const short* tile, int row, int col,
                                       int lane) {
  using lds4 = __attribute__((address_space(3))) half4;
  const short* p = tile + (row + (lane >> 4) * 4 + ((lane & 15) >> 2)) *
                              PITCH + col + (lane & 3) * 4;
  union {
    half4 h[2];
    frag f;
  } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * PITCH));
  return u.f;
}

template <int NA, int NB, int LIMIT>
__device__ __forceinline__ acc4 product(const frag (&a)[NA],
                                        const frag (&b)[NB], acc4 c) {
#pragma unroll
  for (int s = LIMIT; s >= 0; --s)  // small terms first
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0,
                                                    0);
  return c;
}

// Eight values as fragments of N terms.
template <int N>
__device__ __forceinline__ void to_frag(const float (&x)[8], frag (&f)[N]) {
  union {
    unsigned u[4];
    frag f;
  } w[N];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned a[N], b[N];
    cut<N>(x[2 * i], a);
    cut<N>(x[2 * i + 1], b);
#pragma unroll
    for (int n = 0; n < N; ++n) w[n].u[i] = pair(a[n], b[n]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) f[n] = w[n].f;
}

// How rows lie in memory: they begin on 32 bits and are whole vectors of 16
// bytes, more than half of D each, or one of them not more; or they begin and
// end on 32 bits; or neither.
enum Edge { kVectors, kShort, kWords, kHalves };

// The rows of a chunk between global memory and LDS: a thread's part, read
// through a buffer resource that ends with the last row, so that what lies
// behind it reads as zero without a branch, 16 bytes at once from any word.
// Halves are read from the word they begin in and moved by half of it.
// (4 x 2048 tokens, 8 heads of 57 and 79, trained in bf16: 124 us; by single
// elements at the rows' ends, 146 us.  With the tests of words for vectors
// too, 2 x 16384 tokens of heads of 128 take 2% longer.)
template <typename T, int D, int C, Edge EDGE>
struct Rows {
  static constexpr int VE = 16 / sizeof(T);
  static constexpr int kThreads = D * 4;
  static constexpr int N = C * D / VE / kThreads;  // vectors of a thread
  static constexpr int kStep = kThreads / (D / VE);  // rows between them
  union {
    vec<T, VE> v[N];
    vec<unsigned, 4> u[N];
  };
  unsigned more[EDGE == kHalves ? N : 1], shift[EDGE == kHalves ? N : 1];

  // rows at or behind `n` and vectors at or behind `cols` are zero
  __device__ __forceinline__ void read(const T* p, long stride, int n,
                                       int cols) {
    const int row = threadIdx.x / (D / VE);
    const int col = threadIdx.x % (D / VE) * VE;
    const int pitch = int(stride * sizeof(T));
    const int rows = n < C ? n : C;
    const int bytes = (rows - 1) * pitch + cols * (int)sizeof(T);
    if constexpr (EDGE != kHalves) {
      const auto rsrc = buffer(p, bytes);
#pragma unroll
      for (int i = 0; i < N; ++i)
        u[i] = __builtin_amdgcn_raw_buffer_load_b128(
            rsrc, col < cols ? (row + i * kStep) * pitch +
                                   col * (int)sizeof(T)
                             : kBehind, 0, 0);
    } else {
      const int half = int(reinterpret_cast<uintptr_t>(p) & 2);
      const auto rsrc = buffer((const char*)p - half, (bytes + half + 3) & ~3);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = half + (row + i * kStep) * pitch +
                       col * (int)sizeof(T);
        const int word =
            col < cols && row + i * kStep < rows ? at & ~3 : kBehind;
        u[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, word, 0, 0);
        more[i] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, word, 16, 0);
        shift[i] = (at & 2) * 8;
      }
    }
  }

  // What was read of the columns before `cols`, and zero.
  __device__ __forceinline__ vec<unsigned, 4> words(int i, int cols) const {
    vec<unsigned, 4> w = u[i];
    if constexpr (EDGE == kHalves) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        w[d] = __builtin_amdgcn_alignbit(d < 3 ? w[d < 3 ? d + 1 : 3] : more[i],
                                         w[d], shift[i]);
    }
    if (EDGE > kShort && cols % VE) {
      const int col = threadIdx.x % (D / VE) * VE;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int left = cols - col - d * VE / 4;
        w[d] = left >= VE / 4 ? w[d] : left > 0 ? w[d] & 0xffff : 0;
      }
    }
    return w;
  }

  // planes of terms, each C * PITCH
  template <int PITCH, bool LANE_ORDER>
  __device__ __forceinline__ void write(short* tile, int cols) const {
    constexpr int NT = kTerms<T>;
    const int row = threadIdx.x / (D / VE);
    const int col = threadIdx.x % (D / VE) * VE;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      short* dst = tile + (row + i * kStep) * PITCH;
      union {
        vec<unsigned, 4> u;
        vec<T, VE> v;
      } x;
      x.u = words(i, cols);
      unsigned w[NT][VE / 2];
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        if constexpr (NT == 1) {
          w[0][e / 2] = x.u[e / 2];
        } else {
          unsigned a[NT], b[NT];
          cut<NT>(float(x.v[e]), a);
          cut<NT>(float(x.v[e + 1]), b);
#pragma unroll
          for (int n = 0; n < NT; ++n) w[n][e / 2] = pair(a[n], b[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (VE == 8 && !LANE_ORDER) {
          *reinterpret_cast<uint4*>(dst + n * C * PITCH + col) =
              make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]);
        } else {
#pragma unroll
          for (int e = 0; e < VE; e += 4)
            *reinterpret_cast<uint2*>(
                dst + n * C * PITCH +
                (LANE_ORDER ? in_lane_order(col + e) : col + e)) =
                make_uint2(w[n][e / 2], w[n][e / 2 + 1]);
        }
      }
    }
  }
};

// f(0), f(1) .. f(N - 1) with constants.
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>());
  }
}

__device__ __forceinline__ float power(float log2, int n) {
  return __builtin_amdgcn_exp2f(log2 * n);
}

// What a state goes through in n tokens, s lam^n.  While lam^n is above a half
// it is s + s (lam^n - 1): rounded to fp32, a lam^n near one would lose what a
// long memory forgets, the same in each chunk.  Below, lam^n - 1 has lost lam^n
// (at lam^n = 1e-7 all but one bit of it), and the plain product comes before
// a sum with nothing.  Both change the state where it is: with a branch to one
// or the other the compiler copied it behind the products into it, and of the
// ways out of their loop its waits took the longer one for the shorter, so that
// a copy came before the product's result.
struct Decay {
  float by = 0.f, far = 1.f;
  __device__ __forceinline__ void set(float ld, int n) {
    const float x = ld * n;
    const bool near = x > -0.6931f;
    by = near ? expm1f(x) : 0.f;
    far = near ? 1.f : expf(x);
  }
  template <int N>
  __device__ __forceinline__ void operator()(acc4 (&s)[N]) const {
    if (far != 1.f) {
#pragma unroll
      for (int t = 0; t < N; ++t) s[t] *= far;
    }
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[t][r] = __builtin_fmaf(s[t][r], by, s[t][r]);
  }
};

// LDS of a workgroup, in elements of 16 bits.
template <typename T, int D>
struct Lds {
  static constexpr int C = kChunk;
  static constexpr int NT = kTerms<T>, NI = NT == 3 ? 3 : 2;
  static constexpr int kPitch = D + 16;                  // of k and v
  // fp32 at 64 takes smaller pads and three workgroups fit into a CU
  static constexpr int kPitchQ = D == 128 ? 176 : NT == 3 ? 72 : 80;
  static constexpr int kPitchP = D == 64 && NT == 3 ? 40 : 48;
  static constexpr int kTile = C * kPitch, kTileQ = C * kPitchQ;
  static constexpr int kTileP = C * kPitchP;
  static constexpr int kTables = 4 * C;                  // two of C floats
  static constexpr int kState = kTables + 2 * NT * kTile;
  static constexpr int kAll = kState + NT * kTileQ + NI * kTileP;
};

// Waves of a SIMD that registers have to leave room for: as many as LDS does.
template <typename T, int D>
constexpr int kWavesOfUnit = kTerms<T> < 3 ? 4 : D == 64 ? 3 : 2;

// A workgroup takes a segment of a sequence and head for a role; a wave
// keeps 16 columns of the state.  OUT = false computes the state of the
// segment alone.
template <typename T, int D, Edge EDGE, bool OUT>
__global__ __launch_bounds__(D * 4, (kWavesOfUnit<T, D>)) void chunk_kernel(
    Problem pr) {
  using L = Lds<T, D>;
  constexpr int C = kChunk;
  constexpr int kThreads = D * 4, kWaves = D / 16;
  constexpr int NT = L::NT;                // terms of the operands
  constexpr int NI = L::NI;                // of scores and state, as operands
  constexpr int LO = NT == 3 ? 2 : 1;      // that the output needs
  constexpr int KB = D / 32, KT = D / 16;  // blocks and tiles of dk
  constexpr int kTile = L::kTile, kTileQ = L::kTileQ, kTileP = L::kTileP;

  extern __shared__ __attribute__((aligned(16))) short lds[];
  float* const gain = reinterpret_cast<float*>(lds);  // of a token in S
  float* const seen = gain + C;                       // of S at a token
  short* const kt = lds + L::kTables;
  short* const vt = kt + NT * kTile;
  short* const qt = vt + NT * kTile;
  short* const pt = qt + NT * kTileQ;

  // The roles of a problem follow each other on one XCD (workgroups go round
  // the eight of them), where they share what they read in its L2.
  const unsigned turn = blockIdx.x / (8 * pr.roles);
  const unsigned in = blockIdx.x % (8 * pr.roles);
  const unsigned id = turn * 8 + in % 8;
  if (id >= (unsigned)pr.batch * pr.heads * pr.segments) return;
  const Role& ro = pr.role[in / 8];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
  const int seg = id % pr.segments;
  const int bh = id / pr.segments;
  const int b = bh / pr.heads, h = bh % pr.heads;
  const int dk = ro.dk, dv = ro.dv;
  const bool rev = ro.reverse;
  const int entry = rev ? pr.segments - 1 : 0;
  const int exit = rev ? 0 : pr.segments - 1;
  if (!OUT && seg == exit) return;  // nothing comes behind it

  const long len = length_of(pr, b);
  const int seg0 = seg * pr.per_segment;
  const int seg1 = seg0 + pr.per_segment < pr.length
                       ? seg0 + pr.per_segment : pr.length;
  const int live = len < seg1 ? (len > seg0 ? int(len) - seg0 : 0)
                              : seg1 - seg0;  // tokens of the segment
  const int chunks = (live + C - 1) / C;
  const float ld = decay_of(pr, h);
  const float log2 = ld * kLog2e;

  const T* kp = (const T*)ro.k.p + b * ro.k.b + h * ro.k.h + seg0 * ro.k.t;
  const T* vp = (const T*)ro.v.p + b * ro.v.b + h * ro.v.h + seg0 * ro.v.t;
  const T* qp = (const T*)ro.q.p + b * ro.q.b + h * ro.q.h + seg0 * ro.q.t;
  const long ostride = (long)pr.heads * dv;
  T* op = (T*)ro.out;
  if constexpr (OUT)
    op += ((long)b * pr.length + seg0) * ostride + (long)h * dv;

  // chunks on their way to LDS, in registers
  constexpr int kAhead = OUT ? 1 : 2;
  Rows<T, D, C, EDGE> kr[kAhead], vr[kAhead], qr[OUT ? kAhead : 1];
  auto fetch = [&](int step, auto slot) {
    if (step >= chunks) return;
    constexpr int x = decltype(slot)::value;
    const int t0 = (rev ? chunks - 1 - step : step) * C, n = live - t0;
    kr[x].read(kp + t0 * ro.k.t, ro.k.t, n, dk);
    vr[x].read(vp + t0 * ro.v.t, ro.v.t, n, dv);
    if constexpr (OUT) qr[x].read(qp + t0 * ro.q.t, ro.q.t, n, dk);
  };
  each<kAhead>([&](auto slot) { fetch(slot, slot); });

  // the state: tile t has rows 16t + 4g + r of dk, column col0 + l of dv
  const int col0 = wave * 16;
  // Waves behind the last column read and compute scores only.  (Heads of 82
  // and 20, 8 x 2670 tokens, 10 heads, forward in bf16: 101 us -> 90 us.)
  const bool busy = col0 < dv;
  // And the products end with the quarter of D in which the last of dk lies,
  // or with its half.  (16 x 2048 tokens, 8 heads of 64 and 128, trained in
  // bf16: 315 us, 284 us by quarters, 275 us by halves; 2 x 6010 tokens, 11
  // heads of 31 and 117 in fp32: 433 us, 350 us by quarters, 371 us by halves;
  // 4129 tokens of 102 and 96, forward: 115 us -> 120 us.  Whole heads have no
  // such tests, which would cost them 1 to 2%.)
  constexpr int kPart = EDGE == kShort ? D / 2 : D / 4;
  auto behind = [&](int row) {
    return EDGE != kVectors && row % kPart == 0 && row >= dk;
  };
  acc4 s[KT];
  bool some = true;  // whether the state can be other than zero
  float* stored = ro.states + ((long)bh * pr.segments + seg) * (D * D);
  // byte offset of an element of an end's state
  auto offset = [&](int i, int j) {
    const int at = ro.turned ? j * dk + i : i * dv + j;
    return i < dk && j < dv ? at * 4 : kBehind;
  };
  if (seg == entry && ro.first) {
    const auto rsrc = buffer(ro.first + (long)bh * dk * dv, dk * dv * 4);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[t][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            rsrc, offset(t * 16 + 4 * g + r, col0 + l), 0, 0));
  } else if (OUT && seg != entry) {
    if (ro.turned) {  // stored for the transposed state: row and column swap
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[t][r] = stored[wave * (kThreads * 4) + t * 256 + (l >> 2) * 64 +
                           (4 * g + r) * 4 + (l & 3)];
    } else {
#pragma unroll
      for (int t = 0; t < KT; ++t)
        s[t] = *reinterpret_cast<const acc4*>(stored + t * (kThreads * 4) +
                                              threadIdx.x * 4);
    }
  } else {
    some = false;
#pragma unroll
    for (int t = 0; t < KT; ++t) s[t] = acc4{0.f, 0.f, 0.f, 0.f};
  }

  if constexpr (OUT) {
    // the tile of scores that the mask leaves empty is never written again
    for (int i = threadIdx.x; i < NI * kTileP / 2; i += kThreads)
      reinterpret_cast<unsigned*>(pt)[i] = 0;
  }

  Decay decay;
  if constexpr (!OUT) {
    if (some) {
      decay.set(ld, live);
      decay(s);
    }
  }
  // Three waves have a tile of scores each, (0, 0), (1, 1) and the one between
  // them, and the factors of its elements; zero where the mask is.
  const int it = rev ? wave == 1 : wave > 0;
  const int jt = rev ? wave > 0 : wave == 1;
  float fade[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = it * 16 + l, j = jt * 16 + 4 * g + r;
    const int d = rev ? j - i : i - j;
    fade[r] = d >= 0 ? ro.intra * power(log2, d) : 0.f;
  }
  int of_tables = 0;  // the n that tables and `decay` are for
  auto chunk = [&](int step, auto slot) {
    constexpr int x = decltype(slot)::value;
    const int c = rev ? chunks - 1 - step : step;
    const int n = live - c * C < C ? live - c * C : C;
    __syncthreads();  // the last chunk's readers are done
    if constexpr (!OUT) {
      // alone, the state counts decays from the segment's end (backwards in
      // time: from its beginning) and is not touched in between
      const int i = threadIdx.x;
      const int d = rev ? c * C + i + 1 : live - 1 - c * C - i;
      if (i < C) gain[i] = ro.gain * power(log2, d > 0 ? d : 0);
    } else if (n != of_tables) {  // the first chunk, and one not full
      of_tables = n;
      decay.set(ld, n);
      const int i = threadIdx.x % C;
      const int d = rev ? n - 1 - i : i + 1, e = rev ? i + 1 : n - 1 - i;
      if (threadIdx.x < C) gain[i] = ro.gain * power(log2, e > 0 ? e : 0);
      else if (threadIdx.x < 2 * C)
        seen[i] = ro.inter * power(log2, d > 0 ? d : 0);
    }
    kr[x].template write<L::kPitch, false>(kt, dk);
    vr[x].template write<L::kPitch, false>(vt, dv);
    if constexpr (OUT) qr[x].template write<L::kPitchQ, true>(qt, dk);
    fetch(step + kAhead, slot);
    __syncthreads();

    acc4 o[2] = {acc4{0.f, 0.f, 0.f, 0.f}, acc4{0.f, 0.f, 0.f, 0.f}};
    if constexpr (OUT) {
      // scores, transposed: rows j, columns i
      if (wave < 3) {
        acc4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if (behind(kb * 32)) break;
          frag kf[NT], qf[NT];
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            kf[x] = by_row_plain<L::kPitch>(kt + x * kTile, jt * 16, kb * 32,
                                            lane);
            qf[x] = by_row<L::kPitchQ>(qt + x * kTileQ, it * 16, kb * 32,
                                       lane);
          }
          p = product<NT, NT, LO>(kf, qf, p);
        }
        unsigned term[4][NI];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          cut<NI>(fade[r] != 0.f ? p[r] * fade[r] : 0.f, term[r]);
#pragma unroll
        for (int x = 0; x < NI; ++x)
          *reinterpret_cast<uint2*>(
              pt + x * kTileP + (it * 16 + l) * L::kPitchP +
              in_lane_order(jt * 16 + 4 * g)) =
              make_uint2(pair(term[0][x], term[1][x]),
                         pair(term[2][x], term[3][x]));
      }

      // q S, transposed: rows of dv, columns i
      if (some && busy) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if (behind(kb * 32)) break;
          float x[8];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[r] = s[2 * kb][r];
            x[4 + r] = s[2 * kb + 1][r];
          }
          frag sf[NI];
          to_frag<NI>(x, sf);
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            frag qf[NT];
#pragma unroll
            for (int y = 0; y < NT; ++y)
              qf[y] = by_row<L::kPitchQ>(qt + y * kTileQ, it * 16, kb * 32,
                                         lane);
            o[it] = product<NI, NT, LO>(sf, qf, o[it]);
          }
        }
#pragma unroll
        for (int it = 0; it < 2; ++it) o[it] *= seen[it * 16 + l];
      }
      __syncthreads();  // the scores are whole
    }
    if (!busy) return;

    if constexpr (OUT) {
      decay(s);
      some = true;
    }

    frag vf[NT], wf[3];  // v, and v with the weights of its tokens
#pragma unroll
    for (int x = 0; x < NT; ++x)
      vf[x] = by_col<L::kPitch>(vt + x * kTile, 0, col0, lane);
    {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = float(vf[0][e]);
#pragma unroll
        for (int x = 1; x < NT; ++x) y[e] += float(vf[x][e]);
        y[e] *= gain[(e >> 2) * 16 + 4 * g + (e & 3)];
      }
      to_frag<3>(y, wf);
    }
    if constexpr (OUT) {
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        frag pf[NI];
#pragma unroll
        for (int x = 0; x < NI; ++x)
          pf[x] = by_row<L::kPitchP>(pt + x * kTileP, it * 16, 0, lane);
        o[it] = product<NT, NI, LO>(vf, pf, o[it]);
      }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (behind(t * 16)) break;
      frag kf[NT];
#pragma unroll
      for (int x = 0; x < NT; ++x)
        kf[x] = by_col<L::kPitch>(kt + x * kTile, 0, t * 16, lane);
      s[t] = product<NT, 3, 2>(kf, wf, s[t]);
    }

    if constexpr (OUT) {
      const int j = col0 + 4 * g;
      if constexpr (EDGE != kHalves) {
        const int pitch = int(ostride * sizeof(T));
        const auto rsrc = buffer(op + c * C * ostride,
                                 (n - 1) * pitch + dv * (int)sizeof(T));
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const int at = j < dv ? (it * 16 + l) * pitch + j * (int)sizeof(T)
                                : kBehind;
          union {
            vec<T, 4> v;
            vec<unsigned, sizeof(T)> u;
          } r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r.v[e] = T(o[it][e]);
          if (EDGE <= kShort || dv % 4 == 0) {
            if constexpr (sizeof(T) == 2)
              __builtin_amdgcn_raw_buffer_store_b64(r.u, rsrc, at, 0, 0);
            else
              __builtin_amdgcn_raw_buffer_store_b128(r.u, rsrc, at, 0, 0);
          } else {  // the last words of a row are the next one's first
#pragma unroll
            for (int w = 0; w < (int)sizeof(T); ++w)
              __builtin_amdgcn_raw_buffer_store_b32(
                  r.u[w], rsrc,
                  j + w * 4 / (int)sizeof(T) < dv ? at + 4 * w : kBehind, 0,
                  0);
          }
        }
      } else {
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          const int i = it * 16 + l;
          if (i >= n) continue;
          if (j >= dv) continue;
          const float r[4] = {o[it][0], o[it][1], o[it][2], o[it][3]};
          store<T, 4>(op + (c * C + i) * ostride + j, r, dv - j);
        }
      }
    }
  };
  for (int step = 0; step < chunks; step += kAhead)
    each<kAhead>([&](auto slot) {
      if (step + slot < chunks) chunk(step + slot, slot);
    });

  if constexpr (OUT) {
    // behind the sequence's end the output is zero
    for (int i = live + wave; i < seg1 - seg0; i += kWaves)
      for (int j = lane; j < dv; j += 64) op[i * ostride + j] = T(0.f);
    if (seg == exit && ro.last) {
      const auto rsrc = buffer(ro.last + (long)bh * dk * dv, dk * dv * 4);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          __builtin_amdgcn_raw_buffer_store_b32(
              __float_as_uint(s[t][r]), rsrc,
              offset(t * 16 + 4 * g + r, col0 + l), 0, 0);
    }
  } else {
#pragma unroll
    for (int t = 0; t < KT; ++t)
      *reinterpret_cast<acc4*>(stored + t * (kThreads * 4) +
                               threadIdx.x * 4) = s[t];
  }
}

// The state of each segment alone becomes the state that comes into it, for
// the first role.  A thread has four elements of them all; the loads of 16
// segments are in flight at once.  grid: (elements / 1024, batch * heads).
__global__ __launch_bounds__(kThreads) void join_kernel(Problem pr,
                                                        int elements) {
  const int bh = blockIdx.y, b = bh / pr.heads;
  const Role& ro = pr.role[0];
  const long len = length_of(pr, b);
  const float ld = decay_of(pr, bh % pr.heads);
  float* p = ro.states + (long)bh * pr.segments * elements +
             (blockIdx.x * kThreads + threadIdx.x) * 4;
  acc4 carry[1] = {};
  int of = -1;
  Decay decay;
  constexpr int U = 16;
  for (int i0 = 0; i0 < pr.segments; i0 += U) {
    acc4 own[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u < pr.segments ? i0 + u : pr.segments - 1;
      const int seg = ro.reverse ? pr.segments - 1 - i : i;
      own[u] = *reinterpret_cast<const acc4*>(p + (long)seg * elements);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u, seg = ro.reverse ? pr.segments - 1 - i : i;
      if (i < pr.segments) {
        // the entry's own state holds what came in; the exit's is not
        // computed, nor used
        if (i > 0)
          *reinterpret_cast<acc4*>(p + (long)seg * elements) = carry[0];
        const long left = len - (long)seg * pr.per_segment;
        const int n = left < 0 ? 0
                      : left < pr.per_segment ? int(left) : pr.per_segment;
        if (n != of) decay.set(ld, n);
        of = n;
        decay(carry);
        carry[0] += own[u];
      }
    }
  }
}

// One token: the state is read, updated in place and written, and bounds the
// kernel (64 sequences, 16 heads of 64: 7.8 us, 4.4 TB/s).  A workgroup has
// 16 * VE columns of the state of a sequence and head; a thread has VE of
// them in every 16th row.
template <typename T, int VE>
__global__ __launch_bounds__(kThreads) void step_kernel(
    const T* __restrict__ q, const T* __restrict__ k,
    const T* __restrict__ v, float* __restrict__ state, T* __restrict__ o,
    const float* __restrict__ log_decay, int heads, int dk, int dv, long qb,
    long qh, long kb, long kh, long vb, long vh, float scale) {
  __shared__ float sq[128], sk[128];
  __shared__ float part[4][16 * VE];
  const int bh = blockIdx.x, b = bh / heads, h = bh % heads;
  const int t = threadIdx.x;
  if (t < 128) {
    sq[t] = t < dk ? float(q[b * qb + h * qh + t]) * scale : 0.f;
  } else {
    const int i = t - 128;
    sk[i] = i < dk ? float(k[b * kb + h * kh + i]) : 0.f;
  }
  // as in the chunks: a state of a long memory changes by what it forgets
  Decay decay;
  decay.set(log_decay[h], 1);
  const bool near = decay.far == 1.f;
  const float by = near ? decay.by : decay.far;
  const int c = (blockIdx.y * 16 + (t & 15)) * VE;
  const bool on = c < dv;
  float* s = state + (long)bh * dk * dv + c;
  float x[VE], acc[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    x[e] = on ? float(v[b * vb + h * vh + c + e]) : 0.f;
    acc[e] = 0.f;
  }
  __syncthreads();
  if (on) {
#pragma unroll 8
    for (int i = t >> 4; i < dk; i += 16) {
      float r[VE];
      load<float, VE>(s + (long)i * dv, r);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        r[e] = __builtin_fmaf(r[e], by,
                              __builtin_fmaf(sk[i], x[e], near ? r[e] : 0.f));
        acc[e] += sq[i] * r[e];
      }
      store<float, VE>(s + (long)i * dv, r);
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    acc[e] += __shfl_xor(acc[e], 16, 64);
    acc[e] += __shfl_xor(acc[e], 32, 64);
    if ((t & 63) < 16) part[t >> 6][(t & 15) * VE + e] = acc[e];
  }
  __syncthreads();
  if (t < 16 * VE) {
    const int j = blockIdx.y * 16 * VE + t;
    if (j < dv)
      o[(long)bh * dv + j] =
          T(part[0][t] + part[1][t] + part[2][t] + part[3][t]);
  }
}

void check_operand(const torch::Tensor& x, const torch::Tensor& like,
                   int dims, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device() &&
              x.scalar_type() == like.scalar_type() && x.dim() == dims,
              "linear_attention: ", name, " must have ", dims,
              " axes and q's type and GPU");
  for (int i = 0; i + 1 < dims; ++i)
    TORCH_CHECK(x.size(i) == like.size(i), "linear_attention: ", name,
                " differs from q in axis ", i);
  TORCH_CHECK(x.size(dims - 1) >= 1 && x.size(dims - 1) <= 128,
              "linear_attention: heads of 1 to 128 elements, not ",
              x.size(dims - 1));
}

void check_decay(const torch::Tensor& d, const torch::Tensor& q, long heads) {
  TORCH_CHECK(d.is_cuda() && d.device() == q.device() &&
              d.scalar_type() == at::kFloat && d.dim() == 1 &&
              d.size(0) == heads && d.is_contiguous(),
              "linear_attention: log_decay is a contiguous float32 vector "
              "with an element for each head, on q's GPU");
}

void check_state(const torch::Tensor& s, const torch::Tensor& q, long b,
                 long h, long dk, long dv) {
  TORCH_CHECK(s.is_cuda() && s.device() == q.device() &&
              s.scalar_type() == at::kFloat && s.is_contiguous() &&
              s.dim() == 4 && s.size(0) == b && s.size(1) == h &&
              s.size(2) == dk && s.size(3) == dv,
              "linear_attention: a state is float32, contiguous, [batch, "
              "heads, dk, dv], on q's GPU");
}

// contiguous in the last axis
torch::Tensor rows_of(const torch::Tensor& x) {
  return x.stride(-1) == 1 || x.size(-1) == 1 ? x : x.contiguous();
}

// And with tokens that are not on top of each other, nor so far apart that a
// chunk of them exceeds a buffer resource.
torch::Tensor tokens_of(const torch::Tensor& x) {
  const long t = x.stride(1);
  return x.size(1) == 1 || (t >= x.size(3) && t < (1l << 24))
             ? rows_of(x) : x.contiguous();
}

Edge edge_of(const torch::Tensor& x) {
  const int size = (int)x.element_size();
  bool words = reinterpret_cast<uintptr_t>(x.data_ptr()) % 4 == 0 &&
               x.size(-1) * size % 4 == 0;
  for (int i = 0; i + 1 < x.dim(); ++i)
    words = words && (x.size(i) == 1 || x.stride(i) * size % 4 == 0);
  return !words ? kHalves : x.size(-1) * size % 16 ? kWords : kVectors;
}

Operand operand(const torch::Tensor& x) {
  // the stride of an axis of one element can be anything
  return Operand{x.data_ptr(), x.stride(0),
                 x.size(1) == 1 ? x.size(3) : x.stride(1), x.stride(2)};
}

// The lengths of segments: 2 chunks and more where there are 8 of them (546
// tokens, 8 heads, forward: 21 us, with 4 and more 27 us; 256 tokens, 16 heads:
// 20 us both in one segment and in four), as long as there are no more than
// 2048 waves, eight on each CU; more of them cost more in joining states than
// they gain.  (2 x 16384 tokens, 8 heads of 128, trained: 342 us, and 352 us
// with twice as many; 4 x 2048, 16 heads of 64: 160 us, and 174 us with half.)
// A call and its backward pass cut alike.
struct Cut {
  int d, segments, per_segment;
  Cut(const torch::Tensor& q, const torch::Tensor& v) {
    d = q.size(3) <= 64 && v.size(3) <= 64 ? 64 : 128;
    const long alone = q.size(0) * q.size(2);
    const long chunks = (q.size(1) + kChunk - 1) / kChunk;
    const long most = chunks >= 8 ? chunks / 2 : 1;
    const long n = std::max(1l, std::min(32768 / d / alone, most));
    const long per = std::max(1l, (chunks + n - 1) / n);
    per_segment = int(per * kChunk);
    segments = std::max(1, int((chunks + per - 1) / per));
  }
  long states(const torch::Tensor& q) const {
    return segments > 1 ? q.size(0) * q.size(2) * segments * d * d : 0;
  }
};

Edge edge_of_heads(long dk, long dv, const Cut& cut) {
  return std::min(dk, dv) <= cut.d / 2 ? kShort : kVectors;
}

template <typename T, int D, Edge EDGE>
void run_chunks(const Problem& pr, bool state) {
  const long problems = (long)pr.batch * pr.heads * pr.segments;
  const dim3 grid((problems + 7) / 8 * 8 * pr.roles);
  if (state) {
    chunk_kernel<T, D, EDGE, false>
        <<<grid, dim3(D * 4), Lds<T, D>::kState * 2, stream()>>>(pr);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    join_kernel<<<dim3(D * D / (kThreads * 4), pr.batch * pr.heads),
                  dim3(kThreads), 0, stream()>>>(pr, D * D);
  } else {
    constexpr int lds = Lds<T, D>::kAll * 2;
    auto kernel = chunk_kernel<T, D, EDGE, true>;
    // above 64 KB a workgroup has to ask
    if (lds > 65536)
      C10_HIP_CHECK(hipFuncSetAttribute(
          (const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
          lds));
    kernel<<<grid, dim3(D * 4), lds, stream()>>>(pr);
  }
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// The states of the first role's segments where `state`, and otherwise the
// outputs of all roles.
void run_roles(const Problem& pr, const Cut& cut, Edge edge,
               at::ScalarType t, bool state) {
  dispatch(t, "linear_attention", [&](auto x) {
    using T = decltype(x);
    auto go = [&](auto e) {
      if (cut.d == 64) run_chunks<T, 64, decltype(e)::value>(pr, state);
      else run_chunks<T, 128, decltype(e)::value>(pr, state);
    };
    if constexpr (sizeof(T) == 2)
      if (edge == kHalves)
        return go(std::integral_constant<Edge, kHalves>());
    if (edge == kVectors) go(std::integral_constant<Edge, kVectors>());
    else if (edge == kShort) go(std::integral_constant<Edge, kShort>());
    else go(std::integral_constant<Edge, kWords>());
  });
}

Problem problem(const torch::Tensor& q, const torch::Tensor& log_decay,
                const c10::optional<torch::Tensor>& lengths, const Cut& cut) {
  Problem pr{};
  // three roles of 512 threads each stay below the 2^32 of a launch
  TORCH_CHECK(q.size(1) < (1l << 30) && q.size(0) * q.size(2) < (1l << 21),
              "linear_attention: fewer than 2^30 tokens of a sequence and "
              "2^21 sequences times heads");
  TORCH_CHECK(q.size(2) < (1l << 17), "linear_attention: fewer than 2^17 "
              "heads");
  pr.batch = (int)q.size(0);
  pr.length = (int)q.size(1);
  pr.heads = (int)q.size(2);
  pr.segments = cut.segments;
  pr.per_segment = cut.per_segment;
  pr.log_decay = log_decay.data_ptr<float>();
  if (lengths) {
    TORCH_CHECK(lengths->is_cuda() && lengths->device() == q.device() &&
                lengths->dim() == 1 && lengths->size(0) == q.size(0) &&
                lengths->is_contiguous() &&
                (lengths->scalar_type() == at::kLong ||
                 lengths->scalar_type() == at::kInt),
                "linear_attention: lengths is a contiguous vector of int32 "
                "or int64 with an element for each sequence, on q's GPU");
    pr.lengths = lengths->data_ptr();
    pr.long_lengths = lengths->scalar_type() == at::kLong;
  }
  return pr;
}

}  // namespace

// (o, the state behind the sequences, the states before their segments) of
// q, k [batch, length, heads, dk] and v [batch, length, heads, dv].  The
// segments' states are for the backward pass, at most 16 MB.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> linear_attention_fwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v,
    torch::Tensor log_decay, c10::optional<torch::Tensor> first,
    c10::optional<torch::Tensor> lengths, double scale) {
  check_operand(q, q, 4, "q");
  check_operand(k, q, 4, "k");
  check_operand(v, q, 4, "v");
  TORCH_CHECK(q.size(3) == k.size(3), "linear_attention: q and k differ in "
              "their last axis");
  check_decay(log_decay, q, q.size(2));
  const c10::DeviceGuard guard(q.device());
  const long b = q.size(0), h = q.size(2), dk = q.size(3), dv = v.size(3);
  if (first) check_state(*first, q, b, h, dk, dv);
  q = tokens_of(q);
  k = tokens_of(k);
  v = tokens_of(v);
  const auto floats = q.options().dtype(at::kFloat);
  auto o = torch::empty({b, q.size(1), h, dv}, q.options());
  auto last = torch::empty({b, h, dk, dv}, floats);
  if (b * h == 0) return {o, last, torch::empty({0}, floats)};
  const Cut cut(q, v);
  auto states = torch::empty({cut.states(q)}, floats);
  Problem pr = problem(q, log_decay, lengths, cut);
  pr.roles = 1;
  Role& r = pr.role[0];
  r.q = operand(q);
  r.k = operand(k);
  r.v = operand(v);
  r.out = o.data_ptr();
  r.first = first ? first->data_ptr<float>() : nullptr;
  r.last = last.data_ptr<float>();
  r.states = states.data_ptr<float>();
  r.dk = (int)dk;
  r.dv = (int)dv;
  r.intra = r.inter = (float)scale;
  r.gain = 1.f;
  const Edge edge = std::max({edge_of(q), edge_of(k), edge_of(v),
                              edge_of_heads(dk, dv, cut)});
  if (cut.segments > 1) run_roles(pr, cut, edge, q.scalar_type(), true);
  run_roles(pr, cut, edge, q.scalar_type(), false);
  return {o, last, states};
}

// (dq, dk, dv, dfirst) of the gradients of o and of the last state; those
// that are not needed are not computed, and dfirst is empty then.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
linear_attention_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                     torch::Tensor log_decay,
                     c10::optional<torch::Tensor> first,
                     c10::optional<torch::Tensor> lengths, double scale,
                     torch::Tensor states, torch::Tensor go,
                     c10::optional<torch::Tensor> glast, bool need_q,
                     bool need_k, bool need_v, bool need_first) {
  check_operand(q, q, 4, "q");
  check_operand(k, q, 4, "k");
  check_operand(v, q, 4, "v");
  check_operand(go, v, 4, "the output's gradient");
  TORCH_CHECK(q.size(3) == k.size(3) && go.size(3) == v.size(3),
              "linear_attention: last axes differ");
  check_decay(log_decay, q, q.size(2));
  const c10::DeviceGuard guard(q.device());
  const long b = q.size(0), h = q.size(2), dk = q.size(3), dv = v.size(3);
  if (first) check_state(*first, q, b, h, dk, dv);
  if (glast) check_state(*glast, q, b, h, dk, dv);
  q = tokens_of(q);
  k = tokens_of(k);
  v = tokens_of(v);
  go = tokens_of(go);
  const auto floats = q.options().dtype(at::kFloat);
  auto gq = torch::empty(q.sizes(), q.options());
  auto gk = torch::empty(k.sizes(), k.options());
  auto gv = torch::empty(v.sizes(), v.options());
  need_first = need_first && first;
  auto gfirst = torch::empty({need_first ? b : 0, h, dk, dv}, floats);
  if (b * h == 0) return {gq, gk, gv, gfirst};
  const Cut cut(q, v);
  TORCH_CHECK(states.numel() == cut.states(q) && states.is_contiguous() &&
              states.device() == q.device() &&
              states.scalar_type() == at::kFloat,
              "linear_attention: states of another call");
  auto gstates = torch::empty({cut.states(q)}, floats);
  const Edge edge = std::max({edge_of(q), edge_of(k), edge_of(v), edge_of(go),
                              edge_of_heads(dk, dv, cut)});
  const float c = (float)scale;
  Problem pr = problem(q, log_decay, lengths, cut);
  Role e{};  // dv = k G
  e.q = operand(k);
  e.k = operand(q);
  e.v = operand(go);
  e.out = gv.data_ptr();
  e.first = glast ? glast->data_ptr<float>() : nullptr;
  e.last = need_first ? gfirst.data_ptr<float>() : nullptr;
  e.states = gstates.data_ptr<float>();
  e.dk = (int)dk;
  e.dv = (int)dv;
  e.reverse = true;
  e.intra = e.gain = c;
  e.inter = 1.f;
  Role f = e;  // dk = v G^T
  f.q = operand(v);
  f.k = operand(go);
  f.v = operand(q);
  f.out = gk.data_ptr();
  f.last = nullptr;
  f.dk = (int)dv;
  f.dv = (int)dk;
  f.turned = true;
  Role a = f;  // dq = c do S^T
  a.q = operand(go);
  a.k = operand(v);
  a.v = operand(k);
  a.out = gq.data_ptr();
  a.first = first ? first->data_ptr<float>() : nullptr;
  a.states = states.data_ptr<float>();
  a.reverse = false;
  a.inter = c;
  a.gain = 1.f;
  // the states before segments are those of the first role
  const bool backwards = need_k || need_v || need_first;
  if (cut.segments > 1 && backwards) {
    pr.roles = 1;
    pr.role[0] = e;
    run_roles(pr, cut, edge, q.scalar_type(), true);
  }
  pr.roles = 0;
  if (need_v || need_first) pr.role[pr.roles++] = e;
  if (need_k) pr.role[pr.roles++] = f;
  if (need_q) pr.role[pr.roles++] = a;
  if (pr.roles) run_roles(pr, cut, edge, q.scalar_type(), false);
  return {gq, gk, gv, gfirst};
}

// o of one token; the state is updated in place.
torch::Tensor linear_attention_step(torch::Tensor q, torch::Tensor k,
                                    torch::Tensor v, torch::Tensor state,
                                    torch::Tensor log_decay, double scale) {
  check_operand(q, q, 3, "q");
  check_operand(k, q, 3, "k");
  check_operand(v, q, 3, "v");
  TORCH_CHECK(q.size(2) == k.size(2), "linear_attention: q and k differ in "
              "their last axis");
  check_decay(log_decay, q, q.size(1));
  const c10::DeviceGuard guard(q.device());
  const long b = q.size(0), h = q.size(1), dk = q.size(2), dv = v.size(2);
  check_state(state, q, b, h, dk, dv);
  q = rows_of(q);
  k = rows_of(k);
  v = rows_of(v);
  auto o = torch::empty({b, h, dv}, q.options());
  if (b * h == 0) return o;
  check_grid(b * h, kThreads, "linear_attention_step");
  state.unsafeGetTensorImpl()->bump_version();
  // rows of other lengths by elements: heads of 63 take 8.7 us where 64 take
  // 6.8 us, of 127 43 us where 128 take 23 us (64 sequences, 16 heads, bf16,
  // by a graph)
  const bool wide = dv % 4 == 0;
  dispatch(q.scalar_type(), "linear_attention_step", [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto width) {
      constexpr int VE = decltype(width)::value;
      step_kernel<T, VE>
          <<<dim3(b * h, (dv + 16 * VE - 1) / (16 * VE)), dim3(kThreads), 0,
             stream()>>>((const T*)q.data_ptr(), (const T*)k.data_ptr(),
                         (const T*)v.data_ptr(), state.data_ptr<float>(),
                         (T*)o.data_ptr(), log_decay.data_ptr<float>(),
                         (int)h, (int)dk, (int)dv, q.stride(0), q.stride(1),
                         k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                         (float)scale);
    };
    if (wide) go(std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 1>());
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return o;
}

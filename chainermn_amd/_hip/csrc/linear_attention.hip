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
// Long sequences and few heads: the length is cut into segments.  The states
// of the segments alone come first, a scan joins them, and the same kernel
// then starts every segment from its own state.
//
// All products run on bf16 matrix instructions (16x16x32) with fp32 sums:
// a value is cut into terms of 8 bits of mantissa each, exactly: bf16 is one
// term, fp16 two, fp32 three, and products of terms below 2^-24 of the
// largest (2^-16 where the result is rounded to 16 bits) are left out.  The
// state is fp32 throughout, and what is added to it is a product of three
// terms.  The contraction index of a matrix instruction may be permuted if
// both operands are, so that the accumulators of the state and the scores
// (four consecutive rows for a lane) are operands of the next product as
// they stand: lane group g holds 4g..4g+3 and 16+4g..16+4g+3 of 32.

#include "seq_common.h"

namespace {

using namespace seq;

using frag = vec<bf16, 8>;
using acc4 = vec<float, 4>;
using half4 = vec<short, 4>;

constexpr int kThreads = 256;
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
  float first_scale, last_scale;
  int dk, dv;          // of this role
  bool state_by_v;     // the states' rows are this role's v index
  bool reverse;
  bool wide;           // operands can be read by 16 bytes
  float intra, inter, gain;  // factors of scores, q S, and k^T v
};

struct Problem {
  Role role[3];
  const float* log_decay;
  const void* lengths;  // or null
  bool long_lengths;
  int batch, length, heads;
  int segments, per_segment;  // tokens of a segment, a multiple of a chunk
  float* states;  // [role][batch * heads][segments][D * D], in lane order
};

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
template <>
constexpr int kTerms<fp16> = 2;

// Terms are cut off, not rounded: each is exact in bf16, and three of them
// are the whole of an fp32.
template <int N>
__device__ __forceinline__ void cut(float x, unsigned (&term)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned top = __float_as_uint(x) & 0xffff0000u;
    term[i] = top;
    if (i + 1 < N) x -= __uint_as_float(top);
  }
}

// The upper halves of two words, a below b.
__device__ __forceinline__ unsigned pair(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302);
}

// A row-major tile of bf16 in LDS, rows of N elements.  Pieces of 32 bytes
// are permuted within a row by the row's number, so that the 16 rows that a
// fragment reads fall on all banks.
template <int N>
__device__ __forceinline__ int place(int row, int col) {
  static_assert(N == 32 || N == 64 || N == 128, "row length");
  constexpr int shift = N == 128 ? 0 : N == 64 ? 1 : 2;
  constexpr int mask = N / 16 - 1;
  return row * N + (col ^ (((row >> shift) & mask) << 4));
}

// Fragment of 16 rows from `row`, 32 columns from `col`.
template <int N>
__device__ __forceinline__ frag by_row(const short* tile, int row, int col,
                                       int lane) {
  const int r = row + (lane & 15), c = col + (lane >> 4) * 4;
  union {
    half4 h[2];
    frag f;
  } u;
  u.h[0] = *reinterpret_cast<const half4*>(tile + place<N>(r, c));
  u.h[1] = *reinterpret_cast<const half4*>(tile + place<N>(r, c + 16));
  return u.f;
}

// Fragment of 16 columns from `col`, 32 rows from `row`: the transposing
// read gives a lane four rows of one column.
template <int N>
__device__ __forceinline__ frag by_col(const short* tile, int row, int col,
                                       int lane) {
  using lds4 = __attribute__((address_space(3))) half4;
  const int r = row + (lane >> 4) * 4 + ((lane & 15) >> 2);
  const int c = col + (lane & 3) * 4;
  union {
    half4 h[2];
    frag f;
  } u;
  u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds4*)(tile + place<N>(r, c)));
  u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds4*)(tile + place<N>(r + 16, c)));
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

// The rows of a chunk between global memory and LDS: a thread's part.
template <typename T, int D, int C>
struct Rows {
  static constexpr int VE = 16 / sizeof(T);
  static constexpr int N = C * D / VE / kThreads;  // vectors of a thread
  vec<T, VE> v[N];

  // rows at or behind `n` and columns at or behind `cols` are zero
  __device__ __forceinline__ void read(const T* p, long stride, int n,
                                       int cols, bool wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * kThreads + threadIdx.x;
      const int row = at / (D / VE), col = at % (D / VE) * VE;
      const T* src = p + row * stride + col;
      if (wide) {
        if (row < n && col < cols) {
          v[i] = *reinterpret_cast<const vec<T, VE>*>(src);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) v[i][e] = T(0.f);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          v[i][e] = row < n && col + e < cols ? src[e] : T(0.f);
      }
    }
  }

  // planes of terms, each C * D
  __device__ __forceinline__ void write(short* tile) const {
    constexpr int NT = kTerms<T>;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * kThreads + threadIdx.x;
      const int row = at / (D / VE), col = at % (D / VE) * VE;
      short* dst = tile + place<D>(row, col);
      if constexpr (NT == 1) {
        *reinterpret_cast<vec<T, VE>*>(dst) = v[i];
      } else {
        unsigned w[NT][VE / 2];
#pragma unroll
        for (int e = 0; e < VE; e += 2) {
          unsigned a[NT], b[NT];
          cut<NT>(float(v[i][e]), a);
          cut<NT>(float(v[i][e + 1]), b);
#pragma unroll
          for (int n = 0; n < NT; ++n) w[n][e / 2] = pair(a[n], b[n]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (VE == 8)
            *reinterpret_cast<uint4*>(dst + n * C * D) =
                make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]);
          else
            *reinterpret_cast<uint2*>(dst + n * C * D) =
                make_uint2(w[n][0], w[n][1]);
        }
      }
    }
  }
};

__device__ __forceinline__ float power(float log2, int n) {
  return __builtin_amdgcn_exp2f(log2 * n);
}

// A workgroup takes a segment of a sequence and head for a role; a wave
// keeps the state's columns of a quarter of dv.  OUT = false computes the
// state of the segment alone.
template <typename T, int D, int C, bool OUT>
__global__ __launch_bounds__(kThreads, 2) void chunk_kernel(Problem pr) {
  constexpr int NT = kTerms<T>;            // of the operands
  constexpr int NI = NT == 3 ? 3 : 2;      // of scores and state, as operands
  constexpr int LO = NT == 3 ? 2 : 1;      // terms that the output needs
  constexpr int KB = D / 32, KT = D / 16;  // blocks and tiles of dk
  constexpr int W = D / 64;                // tiles of dv of a wave
  constexpr int CT = C / 16, CB = C / 32;  // tiles and blocks of the chunk
  constexpr int kTile = C * D;

  extern __shared__ __attribute__((aligned(16))) short lds[];
  short* const kt = lds;
  short* const vt = kt + NT * kTile;
  short* const qt = vt + NT * kTile;
  short* const pt = qt + (OUT ? NT * kTile : 0);  // scores, NI planes

  const Role& ro = pr.role[blockIdx.y];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, l = lane & 15;
  const int seg = blockIdx.x % pr.segments;
  const int bh = blockIdx.x / pr.segments;
  const int b = bh / pr.heads, h = bh % pr.heads;
  const int dk = ro.dk, dv = ro.dv;
  const bool rev = ro.reverse;
  const int entry = rev ? pr.segments - 1 : 0;
  const int exit = rev ? 0 : pr.segments - 1;
  if (!OUT && seg == exit) return;  // nothing comes behind it

  long len = pr.length;
  if (pr.lengths) {
    const long n = pr.long_lengths ? ((const long*)pr.lengths)[b]
                                   : ((const int*)pr.lengths)[b];
    len = n < 0 ? 0 : n < len ? n : len;
  }
  const int seg0 = seg * pr.per_segment;
  const int seg1 = seg0 + pr.per_segment < pr.length
                       ? seg0 + pr.per_segment : pr.length;
  const int live = len < seg1 ? (len > seg0 ? int(len) - seg0 : 0)
                              : seg1 - seg0;  // tokens of the segment
  const int chunks = (live + C - 1) / C;

  // exp(-200) is zero in fp32, and 0 * log2 has to be 0; NaN stays
  float ld = pr.log_decay[h];
  ld = ld < -200.f ? -200.f : ld;
  const float log2 = ld * kLog2e;

  const T* kp = (const T*)ro.k.p + b * ro.k.b + h * ro.k.h + seg0 * ro.k.t;
  const T* vp = (const T*)ro.v.p + b * ro.v.b + h * ro.v.h + seg0 * ro.v.t;
  const T* qp = (const T*)ro.q.p + b * ro.q.b + h * ro.q.h + seg0 * ro.q.t;
  T* op = (T*)ro.out;
  long ostride = 0;
  if constexpr (OUT) {
    ostride = (long)pr.heads * dv;
    op += ((long)b * pr.length + seg0) * ostride + (long)h * dv;
  }

  // the state: tile t has rows 16t + 4g + r of dk, column l of dv tile w
  acc4 s[KT][W];
  float* mine = nullptr;
  if (pr.states)
    mine = pr.states + (((long)blockIdx.y * pr.batch * pr.heads + bh) *
                            pr.segments + seg) * (D * D) + threadIdx.x * 4;
  const int col0 = wave * W * 16;
  bool some = false;  // whether the state can be other than zero
  if (seg == entry) {
    some = ro.first != nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = t * 16 + 4 * g + r, j = col0 + w * 16 + l;
          s[t][w][r] = some && i < dk && j < dv
              ? ro.first[(long)bh * dk * dv +
                         (ro.state_by_v ? (long)j * dk + i
                                        : (long)i * dv + j)] * ro.first_scale
              : 0.f;
        }
  } else if (OUT) {
    some = true;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int w = 0; w < W; ++w)
        s[t][w] = *reinterpret_cast<const acc4*>(
            mine + (t * W + w) * (kThreads * 4));
  } else {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int w = 0; w < W; ++w) s[t][w] = acc4{0.f, 0.f, 0.f, 0.f};
  }

  Rows<T, D, C> kr, vr, qr;
  auto fetch = [&](int c) {
    const int t0 = c * C, n = live - t0;
    kr.read(kp + t0 * ro.k.t, ro.k.t, n, dk, ro.wide);
    vr.read(vp + t0 * ro.v.t, ro.v.t, n, dv, ro.wide);
    if constexpr (OUT) qr.read(qp + t0 * ro.q.t, ro.q.t, n, dk, ro.wide);
  };
  if (chunks > 0) fetch(rev ? chunks - 1 : 0);
  if constexpr (OUT) {
    // tiles of scores that the mask leaves empty are never written again
    for (int i = threadIdx.x; i < NI * C * C / 2; i += kThreads)
      reinterpret_cast<unsigned*>(pt)[i] = 0;
  }

  for (int step = 0; step < chunks; ++step) {
    const int c = rev ? chunks - 1 - step : step;
    const int n = live - c * C < C ? live - c * C : C;
    __syncthreads();  // the last chunk's readers are done
    kr.write(kt);
    vr.write(vt);
    if constexpr (OUT) qr.write(qt);
    if (step + 1 < chunks) fetch(rev ? c - 1 : c + 1);
    __syncthreads();

    acc4 o[CT][W];
    if constexpr (OUT) {
      // scores, transposed: rows j, columns i
      for (int e = wave; e < CT * (CT + 1) / 2; e += 4) {
        const int hi = e < 1 ? 0 : e < 3 ? 1 : e < 6 ? 2 : 3;
        const int lo = e - hi * (hi + 1) / 2;
        const int it = rev ? lo : hi, jt = rev ? hi : lo;
        acc4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          frag kf[NT], qf[NT];
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            kf[x] = by_row<D>(kt + x * kTile, jt * 16, kb * 32, lane);
            qf[x] = by_row<D>(qt + x * kTile, it * 16, kb * 32, lane);
          }
          p = product<NT, NT, LO>(kf, qf, p);
        }
        unsigned term[4][NI];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = it * 16 + l, j = jt * 16 + 4 * g + r;
          const int d = rev ? j - i : i - j;
          const float x = d >= 0 ? p[r] * (ro.intra * power(log2, d)) : 0.f;
          cut<NI>(x, term[r]);
        }
#pragma unroll
        for (int x = 0; x < NI; ++x)
          *reinterpret_cast<uint2*>(
              pt + x * C * C + place<C>(it * 16 + l, jt * 16 + 4 * g)) =
              make_uint2(pair(term[0][x], term[1][x]),
                         pair(term[2][x], term[3][x]));
      }

      // q S, transposed: rows of dv, columns i
#pragma unroll
      for (int it = 0; it < CT; ++it)
#pragma unroll
        for (int w = 0; w < W; ++w) o[it][w] = acc4{0.f, 0.f, 0.f, 0.f};
      if (some) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          frag sf[W][NI];
#pragma unroll
          for (int w = 0; w < W; ++w) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              x[r] = s[2 * kb][w][r];
              x[4 + r] = s[2 * kb + 1][w][r];
            }
            to_frag<NI>(x, sf[w]);
          }
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            frag qf[NT];
#pragma unroll
            for (int x = 0; x < NT; ++x)
              qf[x] = by_row<D>(qt + x * kTile, it * 16, kb * 32, lane);
#pragma unroll
            for (int w = 0; w < W; ++w)
              o[it][w] = product<NI, NT, LO>(sf[w], qf, o[it][w]);
          }
        }
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          const int i = it * 16 + l;
          const int d = rev ? n - 1 - i : i + 1;
          const float f = ro.inter * power(log2, d > 0 ? d : 0);
#pragma unroll
          for (int w = 0; w < W; ++w) o[it][w] *= f;
        }
      }
      __syncthreads();  // the scores are whole
    }

    const float less = expm1f(ld * n);  // keeps a decay near one exact
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[t][w][r] = __builtin_fmaf(s[t][w][r], less, s[t][w][r]);

#pragma unroll
    for (int jb = 0; jb < CB; ++jb) {
      float weight[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = jb * 32 + 4 * g + (e & 3) + (e >> 2) * 16;
        const int d = rev ? j + 1 : n - 1 - j;
        weight[e] = ro.gain * power(log2, d > 0 ? d : 0);
      }
      frag vf[W][NT], wf[W][3];
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
          vf[w][x] = by_col<D>(vt + x * kTile, jb * 32, col0 + w * 16, lane);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = float(vf[w][0][e]);
#pragma unroll
          for (int x = 1; x < NT; ++x) y[e] += float(vf[w][x][e]);
          y[e] *= weight[e];
        }
        to_frag<3>(y, wf[w]);
      }
      if constexpr (OUT) {
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          if (rev ? it > 2 * jb + 1 : it < 2 * jb) continue;
          frag pf[NI];
#pragma unroll
          for (int x = 0; x < NI; ++x)
            pf[x] = by_row<C>(pt + x * C * C, it * 16, jb * 32, lane);
#pragma unroll
          for (int w = 0; w < W; ++w)
            o[it][w] = product<NT, NI, LO>(vf[w], pf, o[it][w]);
        }
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        frag kf[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x)
          kf[x] = by_col<D>(kt + x * kTile, jb * 32, t * 16, lane);
#pragma unroll
        for (int w = 0; w < W; ++w)
          s[t][w] = product<NT, 3, 2>(kf, wf[w], s[t][w]);
      }
    }
    some = true;

    if constexpr (OUT) {
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        const int i = it * 16 + l;
        if (i >= n) continue;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int j = col0 + w * 16 + 4 * g;
          T* dst = op + (c * C + i) * ostride + j;
          float r[4] = {o[it][w][0], o[it][w][1], o[it][w][2], o[it][w][3]};
          if (dv % 4 == 0) {
            if (j < dv) store<T, 4>(dst, r);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j + e < dv) dst[e] = T(r[e]);
          }
        }
      }
    }
  }

  if constexpr (OUT) {
    // behind the sequence's end the output is zero
    for (int i = live + threadIdx.x / 64; i < seg1 - seg0; i += kThreads / 64)
      for (int j = lane; j < dv; j += 64) op[i * ostride + j] = T(0.f);
    if (seg == exit && ro.last) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = t * 16 + 4 * g + r, j = col0 + w * 16 + l;
            if (i < dk && j < dv)
              ro.last[(long)bh * dk * dv +
                      (ro.state_by_v ? (long)j * dk + i
                                     : (long)i * dv + j)] =
                  s[t][w][r] * ro.last_scale;
          }
    }
  } else {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int w = 0; w < W; ++w)
        *reinterpret_cast<acc4*>(mine + (t * W + w) * (kThreads * 4)) =
            s[t][w];
  }
}

// The state of each segment alone becomes the state that comes into it.
// grid: (elements / 1024, batch * heads, roles).
__global__ __launch_bounds__(kThreads) void join_kernel(Problem pr,
                                                        int elements) {
  const int bh = blockIdx.y, b = bh / pr.heads, h = bh % pr.heads;
  const bool rev = pr.role[blockIdx.z].reverse;
  long len = pr.length;
  if (pr.lengths) {
    const long n = pr.long_lengths ? ((const long*)pr.lengths)[b]
                                   : ((const int*)pr.lengths)[b];
    len = n < 0 ? 0 : n < len ? n : len;
  }
  float ld = pr.log_decay[h];
  ld = ld < -200.f ? -200.f : ld;
  float* p = pr.states +
             ((long)blockIdx.z * gridDim.y + bh) * pr.segments * elements +
             (blockIdx.x * kThreads + threadIdx.x) * 4;
  acc4 carry = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < pr.segments; ++i) {
    const int seg = rev ? pr.segments - 1 - i : i;
    acc4* at = reinterpret_cast<acc4*>(p + (long)seg * elements);
    // the entry's own state holds what came in; the exit's is not computed
    const acc4 own = i + 1 < pr.segments ? *at : carry;
    if (i > 0) *at = carry;
    const long left = len - (long)seg * pr.per_segment;
    const int n = left < 0 ? 0
                  : left < pr.per_segment ? int(left) : pr.per_segment;
    const float less = expm1f(ld * n);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      carry[r] = __builtin_fmaf(carry[r], less, carry[r]) + own[r];
  }
}

// One token: the state is read, updated in place and written, and bounds the
// kernel.  A workgroup has 16 * VE columns of the state of a sequence and
// head; a thread has VE of them in every 16th row.
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
  const float lam = expf(log_decay[h]);
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
        r[e] = r[e] * lam + sk[i] * x[e];
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

bool is_wide(const torch::Tensor& x) {
  const int ve = 16 / (int)x.element_size();
  bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
            x.size(-1) % ve == 0;
  for (int i = 0; i + 1 < x.dim(); ++i)
    ok = ok && (x.size(i) == 1 || x.stride(i) % ve == 0);
  return ok;
}

Operand operand(const torch::Tensor& x) {
  return Operand{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}

template <typename T, int D, int C>
void run_chunks(Problem& pr, int roles) {
  constexpr int NT = kTerms<T>, NI = NT == 3 ? 3 : 2;
  const int lds_out = (3 * NT * C * D + NI * C * C) * 2;
  const int lds_state = 2 * NT * C * D * 2;
  const dim3 grid(pr.batch * pr.heads * pr.segments, roles);
  if (pr.segments > 1) {
    chunk_kernel<T, D, C, false>
        <<<grid, dim3(kThreads), lds_state, stream()>>>(pr);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    join_kernel<<<dim3(D * D / (kThreads * 4), pr.batch * pr.heads, roles),
                  dim3(kThreads), 0, stream()>>>(pr, D * D);
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  auto kernel = chunk_kernel<T, D, C, true>;
  // above 64 KB a workgroup has to ask
  C10_HIP_CHECK(hipFuncSetAttribute(
      (const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
      lds_out));
  kernel<<<grid, dim3(kThreads), lds_out, stream()>>>(pr);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

void run_roles(Problem& pr, int roles, const torch::Tensor& q,
               const torch::Tensor& log_decay,
               const c10::optional<torch::Tensor>& lengths) {
  pr.batch = (int)q.size(0);
  pr.length = (int)q.size(1);
  pr.heads = (int)q.size(2);
  TORCH_CHECK(q.size(1) < (1l << 30) && q.size(0) * q.size(2) < (1l << 30),
              "linear_attention: fewer than 2^30 tokens of a sequence, and "
              "sequences times heads");
  pr.log_decay = log_decay.data_ptr<float>();
  pr.lengths = nullptr;
  pr.long_lengths = false;
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
  int widest = 0;
  for (int i = 0; i < roles; ++i) {
    widest = std::max(widest, std::max(pr.role[i].dk, pr.role[i].dv));
  }
  const int d = widest <= 64 ? 64 : 128;
  const bool is_bf16 = q.scalar_type() == at::kBFloat16;
  const int chunk = is_bf16 ? 64 : 32;
  // Segments of 4 chunks and more, until two workgroups have work on each
  // of 256 CUs.
  const long alone = (long)pr.batch * pr.heads * roles;
  const long chunks = (pr.length + chunk - 1) / chunk;
  long segments = std::min((512 + alone - 1) / alone, chunks / 4);
  if (segments < 1) segments = 1;
  const long per = std::max(1l, (chunks + segments - 1) / segments);
  pr.per_segment = int(per * chunk);
  pr.segments = int((chunks + per - 1) / per);
  if (pr.segments < 1) pr.segments = 1;
  torch::Tensor space;
  pr.states = nullptr;
  if (pr.segments > 1) {
    space = torch::empty({alone * pr.segments * d * d},
                         q.options().dtype(at::kFloat));
    pr.states = space.data_ptr<float>();
  }
  dispatch(q.scalar_type(), "linear_attention", [&](auto t) {
    using T = decltype(t);
    constexpr int C = sizeof(T) == 2 && std::is_same<T, bf16>::value ? 64
                                                                     : 32;
    if (d == 64) run_chunks<T, 64, C>(pr, roles);
    else run_chunks<T, 128, C>(pr, roles);
  });
}

}  // namespace

// (o, the state behind the sequence) of q, k [batch, length, heads, dk] and
// v [batch, length, heads, dv].
std::tuple<torch::Tensor, torch::Tensor> linear_attention_fwd(
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
  q = rows_of(q);
  k = rows_of(k);
  v = rows_of(v);
  auto o = torch::empty({b, q.size(1), h, dv}, q.options());
  auto last = torch::empty({b, h, dk, dv}, q.options().dtype(at::kFloat));
  if (last.numel() == 0) return {o, last};
  Problem pr{};
  Role& r = pr.role[0];
  r.q = operand(q);
  r.k = operand(k);
  r.v = operand(v);
  r.out = o.data_ptr();
  r.first = first ? first->data_ptr<float>() : nullptr;
  r.last = last.data_ptr<float>();
  r.first_scale = r.last_scale = 1.f;
  r.dk = (int)dk;
  r.dv = (int)dv;
  r.wide = is_wide(q) && is_wide(k) && is_wide(v);
  r.intra = r.inter = (float)scale;
  r.gain = 1.f;
  run_roles(pr, 1, q, log_decay, lengths);
  return {o, last};
}

// (dq, dk, dv, dfirst) of the gradients of o and of the last state; dfirst
// is empty where no state came in.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
linear_attention_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                     torch::Tensor log_decay,
                     c10::optional<torch::Tensor> first,
                     c10::optional<torch::Tensor> lengths, double scale,
                     torch::Tensor go, c10::optional<torch::Tensor> glast) {
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
  q = rows_of(q);
  k = rows_of(k);
  v = rows_of(v);
  go = rows_of(go);
  auto gq = torch::empty(q.sizes(), q.options());
  auto gk = torch::empty(k.sizes(), k.options());
  auto gv = torch::empty(v.sizes(), v.options());
  auto gfirst = torch::empty({first ? b : 0, h, dk, dv},
                             q.options().dtype(at::kFloat));
  if (b * h == 0) return {gq, gk, gv, gfirst};
  Problem pr{};
  const bool wide = is_wide(q) && is_wide(k) && is_wide(v) && is_wide(go);
  const float c = (float)scale;
  Role& a = pr.role[0];  // dq = c do S^T
  a.q = operand(go);
  a.k = operand(v);
  a.v = operand(k);
  a.out = gq.data_ptr();
  a.first = first ? first->data_ptr<float>() : nullptr;
  a.first_scale = 1.f;
  a.dk = (int)dv;
  a.dv = (int)dk;
  a.state_by_v = true;
  a.wide = wide;
  a.intra = a.inter = c;
  a.gain = 1.f;
  Role& e = pr.role[1];  // dv = k G
  e.q = operand(k);
  e.k = operand(q);
  e.v = operand(go);
  e.out = gv.data_ptr();
  e.first = glast ? glast->data_ptr<float>() : nullptr;
  e.first_scale = 1.f;
  e.last = first ? gfirst.data_ptr<float>() : nullptr;
  e.last_scale = 1.f;
  e.dk = (int)dk;
  e.dv = (int)dv;
  e.reverse = true;
  e.wide = wide;
  e.intra = e.gain = c;
  e.inter = 1.f;
  Role& f = pr.role[2];  // dk = v G^T
  f.q = operand(v);
  f.k = operand(go);
  f.v = operand(q);
  f.out = gk.data_ptr();
  f.first = e.first;
  f.first_scale = 1.f;
  f.dk = (int)dv;
  f.dv = (int)dk;
  f.state_by_v = true;
  f.reverse = true;
  f.wide = wide;
  f.intra = f.gain = c;
  f.inter = 1.f;
  run_roles(pr, 3, q, log_decay, lengths);
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
  const int ve = vector_width(state.data_ptr(), dv, dv, 4);
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
    if (ve == 4) go(std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 1>());
  });
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return o;
}

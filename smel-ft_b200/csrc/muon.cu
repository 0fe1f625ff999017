// Orthogonalised updates of LoRA factors: x -> the Newton-Schulz polynomial of x, alone or inside a momentum step.
//
//   X0 = x / (|x|_F + eps);   X <- a X + b (X X^T) X + c (X X^T)^2 X,  `steps` times, on the short side d <= 64.
//
// Every iterate is a polynomial in G0 = X0 X0^T times X0, so the long side is needed only twice: once for the Gram
// matrix and once for the product P X0. Between them, on d x d matrices that commute and are symmetric:
//   S = a I + b G + c G^2;   P <- S P;   G <- S G S.
// Precision. The steps grow a singular value near zero by a^steps (485 for the usual polynomial), and an error delta in
// G moves the result by delta / sigma^2, so gradients of low rank (few tokens reached the expert) come out up to 3e-4
// off when G is held in fp32, and 6e-5 with the last product alone in fp32 (P has entries up to 485 there, and the sums
// cancel them). All of it is fp64, on the fp64 matrix instruction (m8n8k4), and rounded once. An fp32 last product for
// the updates that allow it was built and was no faster (192 x 64 x 2048: 287 us against 275; 512 x 16 x 2048: 69, 64).
// The momentum update itself is rounded to fp32, as its buffer is.
//
// The d x d recurrence never returns to x, so the rounding of G in directions that x barely has grows by a^2 a step: it moves the
// result by up to 0.45 * 2^-53 times the product of the a^2 but the last (restated on the CPU against whole numbers of 260
// bits). Polynomials that let the product pass 2^26 (more than eight steps of the usual one) take careful_kernel, which holds
// sums and d x d matrices in pairs of doubles.
//
// Two ways, by the size of a matrix:
//   resident  a cluster of 1 to 8 blocks holds one matrix in shared memory and reads it once (ortho_kernel)
//   split     many blocks add partial Gram matrices of one matrix, one block forms P, many blocks apply it
//             (gram_kernel, form_kernel, product_kernel); x is read twice
#include <algorithm>
#include <atomic>
#include <memory>
#include <mutex>
#include <new>

#include "common.cuh"
#include "host.h"
#include "smelb.h"

namespace smelb {
namespace {

constexpr int kThreads = 256, kWarps = 8;
// Columns of a chunk of the split way: 16 to 66 KB (512 columns up to 32 rows: 169 us for 300 x 16 x 8192, 335 with 128).
__host__ __device__ constexpr int split_cap(int nt) { return nt <= 4 ? 512 : 128; }
constexpr int kDevErrWaitCluster = 16;  // a block waiting for its cluster's parts of the Gram matrix
constexpr int kMaxSteps = 16, kMaxTensors = 48, kMaxD = 64;

struct Tensor {
  void* p;          // parameter (momentum step) or output
  const void* g;    // gradient or input
  float* m;         // momentum buffer
  long long start;  // split: matrices before this tensor's; resident: clusters
  int batch;        // matrices
  int shift;        // resident: 2^shift blocks of a cluster hold one matrix
  int d, L;         // short and long side
  int tall;         // memory is [L][d] (else [d][L])
  // factors of divisions, 2^32 / n + 1: by d, and by the columns that kThreads vectors of 4 or 8 elements cover at once
  uint32_t by_d, by_jump[2];
  float step;       // lr * shape factor
};

struct Args {
  Tensor t[kMaxTensors];
  int n, steps;
  long long first;   // split: the launch's first matrix
  int blocks;        // split: blocks of one matrix; resident: of a cluster, 2^shift
  int shift;
  int cap;           // columns that a block holds at once (a multiple of 32)
  // wide matrices in vectors of 4 and 8 elements: the rows that the block covers at once (two or more: cap is at most 512),
  // and the factors of divisions by the vectors of a row and by those rows
  int rows[2];
  uint32_t by_v[2], by_rows[2];
  float mu, omu, decay;  // omu: 1 - momentum, from 64 bits
  int nesterov;
  double eps;
  int* err;      // status words
  double* gram;  // split: [matrix][block][PART] partial Gram matrices
  double* form;  // split: [matrix][NT * NT * 64] P
  double coef[kMaxSteps][3];
};

// d x d matrices are NT x NT tiles of 8 x 8 doubles, row-major in the tile, so a lane's two accumulators of the matrix
// instruction (row lane / 4, columns 2 (lane % 4) + e) are 16 bytes at 2 lane. Read with those indices they are also the
// instruction's operands when the sum over k takes the columns in the order 2 c + e (c the lane's place, e the step):
// as the left one directly, as the right one because the matrices are symmetric. A product of tiles is two 16-byte
// loads for two instructions, without a shuffle.
template <int NT>
struct Dims {
  static constexpr int D = NT * 8;
  static constexpr int TILES = NT * (NT + 1) / 2;       // tiles of the upper triangle
  static constexpr int GROUPS = NT == 8 ? 4 : 1;        // tile groups among the warps (accumulators in registers)
  static constexpr int ACC = GROUPS == 1 ? TILES : NT + 1;  // tiles of a group
  static constexpr int KG = kWarps / GROUPS;            // warps that split the columns
  static constexpr int BUFS = NT >= 3 ? 2 : 4;          // the warps' partial Gram matrices in shared memory at once
  static constexpr int MAT = NT * NT * 64;              // doubles of one matrix
  static constexpr int PART = TILES * 64;               // doubles of one packed upper triangle
  static constexpr int POLY = (NT <= 2 ? 5 : 4) * MAT;  // S (two up to 16 rows), V and two P
  // doubles of the work space that S, V and P share with what comes before them: the warps' partial sums, then one
  // from each block of the cluster
  static constexpr int work(int cluster) {
    return POLY > (BUFS + cluster) * PART ? POLY : (BUFS + cluster) * PART;
  }
};

// Pitch of the columns in shared memory: 4 mod 32, so the operands of the Gram product (8 rows x 4 columns) and of the
// product with P (rows 2 c + e, 8 columns) both touch 32 different banks.
__host__ __device__ constexpr int pitch(int cap) { return cap + 4; }

__device__ __forceinline__ void dmma(double (&c)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
      : "+d"(c[0]), "+d"(c[1])
      : "d"(a), "d"(b));
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// 16 bytes into the same place of the cluster's block `rank`, counted by its barrier `bar`.
__device__ __forceinline__ void push(double* to, uint64_t* bar, int rank, double a, double b) {
  uint32_t at, mb;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(to)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(mb) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(at), "d"(a),
               "d"(b), "r"(mb)
               : "memory");
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// The momentum update u of one element from its gradient and buffer; `first` (the buffer is still the old one) renews it.
__device__ __forceinline__ float update(const Args& a, float g, float& m, bool first) {
  if (first) m = fmaf(a.mu, m, a.omu * g);
  return a.nesterov ? fmaf(a.mu, m, a.omu * g) : m;
}

// 16 bytes of T as floats and back.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
};
__device__ __forceinline__ void unpack(const uint4& r, Vec<float>& o) {
  o.v[0] = __uint_as_float(r.x);
  o.v[1] = __uint_as_float(r.y);
  o.v[2] = __uint_as_float(r.z);
  o.v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(const uint4& r, Vec<bf16>& o) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    o.v[2 * k] = __uint_as_float(w[k] << 16);
    o.v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 repack(const Vec<float>& o) {
  return make_uint4(__float_as_uint(o.v[0]), __float_as_uint(o.v[1]), __float_as_uint(o.v[2]), __float_as_uint(o.v[3]));
}
__device__ __forceinline__ uint4 repack(const Vec<bf16>& o) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(o.v[2 * k], o.v[2 * k + 1]);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}


// A thread's vectors of N elements among a block's columns [j0, j0 + w). Its place along the contiguous side is fixed and
// it goes along the other one, so that a vector costs two additions: in a wide matrix [d][L] the thread has the columns
// from N (tid % (cap / N)) of every rows-th row, in a tall one [L][d] N of the d elements of every columns-th column.
template <int N>
struct Walk {
  int n;            // vectors
  int at, step;     // offset in memory from (0, j0), and to the next vector (a matrix has less than 2^31 elements)
  int in, in_step;  // the same in x
  __device__ __forceinline__ Walk(const Args& a, const Tensor& t, int w, int ld) {
    const int tid = threadIdx.x;
    if (t.tall) {
      const int j = (int)__umulhi((uint32_t)(tid * N), t.by_d), i = tid * N - j * t.d;
      const int jump = (int)__umulhi((uint32_t)(kThreads * N), t.by_d);  // columns that the block covers at once
      n = j < jump && j < w ? (int)__umulhi((uint32_t)(w - 1 - j), t.by_jump[N == 8]) + 1 : 0;
      at = tid * N;
      step = jump * t.d;
      in = i * ld + j;
      in_step = jump;
    } else {
      const int i = (int)__umulhi((uint32_t)tid, a.by_v[N == 8]), j = (tid - i * (a.cap / N)) * N;
      const int jump = a.rows[N == 8];  // rows that the block covers at once
      n = i < jump && i < t.d && j < w ? (int)__umulhi((uint32_t)(t.d - 1 - i), a.by_rows[N == 8]) + 1 : 0;
      at = i * t.L + j;
      step = jump * t.L;
      in = i * ld + j;
      in_step = jump * ld;
    }
  }
};

// The N elements of a vector: v -> x (PUT) or x -> v.
template <bool PUT, int N, bool TALL>
__device__ __forceinline__ void move(float* c, int ld, float (&v)[N]) {
  if (TALL) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (PUT) c[k * ld] = v[k];
      else v[k] = c[k * ld];
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      float4* f = reinterpret_cast<float4*>(c + k);
      if (PUT) {
        *f = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else {
        const float4 o = *f;
        v[k] = o.x;
        v[k + 1] = o.y;
        v[k + 2] = o.z;
        v[k + 3] = o.w;
      }
    }
  }
}

// Whether the vectors of a slice start on 16 bytes and end with it.
template <typename T, bool MUON>
__device__ __forceinline__ bool vectors(const Tensor& t, long long base, int w) {
  constexpr int N = 16 / sizeof(T);
  const uintptr_t at = (uintptr_t)(reinterpret_cast<const T*>(t.g) + base) |
                       (uintptr_t)(reinterpret_cast<T*>(t.p) + base) | (MUON ? (uintptr_t)(t.m + base) : 0);
  return (at & 15) == 0 && (t.tall ? t.d % N == 0 : t.L % N == 0 && w % N == 0);
}

template <typename T, bool MUON, bool TALL>
__device__ __forceinline__ void load_vectors(const Args& a, const Tensor& t, const T* g, float* m, int w, float* x,
                                             int ld, bool first) {
  constexpr int N = Vec<T>::N, U = MUON && N == 8 ? 2 : 4;  // vectors in flight per thread
  const Walk<N> walk(a, t, w, ld);
  int at = walk.at;
  float* in = x + walk.in;
  for (int left = walk.n; left > 0; left -= U) {
    uint4 rg[U], rm[U][N / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < left) {
        rg[u] = __ldg(reinterpret_cast<const uint4*>(g + at + u * walk.step));
        if (MUON) {
#pragma unroll
          for (int k = 0; k < N / 4; ++k) rm[u][k] = *reinterpret_cast<const uint4*>(m + at + u * walk.step + 4 * k);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < left) {
        Vec<T> v;
        unpack(rg[u], v);
        if (MUON) {
#pragma unroll
          for (int k = 0; k < N / 4; ++k) {
            Vec<float> b;
            unpack(rm[u][k], b);
#pragma unroll
            for (int l = 0; l < 4; ++l) v.v[4 * k + l] = update(a, v.v[4 * k + l], b.v[l], first);
            if (first) *reinterpret_cast<uint4*>(m + at + u * walk.step + 4 * k) = repack(b);
          }
        }
        move<true, N, TALL>(in + u * walk.in_step, ld, v.v);
      }
    }
    at += U * walk.step;
    in += U * walk.in_step;
  }
}

// Single elements of w columns, for matrices whose rows do not start on 16 bytes: calls f(u, offset in memory, place in x)
// for up to U elements, u < U, between two calls of done(). A warp takes every eighth row of a wide matrix; a tall one is
// contiguous, and a thread's next element is kThreads on.
template <int U, class F, class G>
__device__ __forceinline__ void elements(const Tensor& t, int w, int ld, F&& f, G&& done) {
  if (t.tall) {
    int j = (int)__umulhi((uint32_t)threadIdx.x, t.by_d), i = threadIdx.x - j * t.d;
    const int dj = (int)__umulhi((uint32_t)kThreads, t.by_d), di = kThreads - dj * t.d;
    for (int q = threadIdx.x; q < w * t.d; q += U * kThreads) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q + u * kThreads < w * t.d) f(u, q + u * kThreads, i * ld + j);
        i += di;
        j += dj;
        if (i >= t.d) {
          i -= t.d;
          ++j;
        }
      }
      done();
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < t.d; i += kWarps)
      for (int j = lane; j < w; j += U * 32) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j + u * 32 < w) f(u, i * t.L + j + u * 32, i * ld + j + u * 32);
        done();
      }
  }
}

template <typename T, bool MUON>
__device__ __noinline__ void load_elements(const Args& a, const Tensor& t, const T* g, float* m, int w, float* x, int ld,
                                           bool first) {
  constexpr int U = 8;
  float rg[U], rm[U];
  int at[U], in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) at[u] = -1;
  elements<U>(t, w, ld,
              [&](int u, int from, int to) {
                at[u] = from;
                in[u] = to;
                rg[u] = to_f(g[from]);
                if (MUON) rm[u] = m[from];
              },
              [&] {
#pragma unroll
                for (int u = 0; u < U; ++u)
                  if (at[u] >= 0) {
                    float v = rg[u];
                    if (MUON) {
                      v = update(a, v, rm[u], first);
                      if (first) m[at[u]] = rm[u];
                    }
                    x[in[u]] = v;
                    at[u] = -1;
                  }
              });
}

// The result o at a place whose present value is p.
template <bool MUON>
__device__ __forceinline__ float result(const Args& a, const Tensor& t, float o, float p) {
  return MUON ? fmaf(-t.step, o, p * a.decay) : o;
}

template <typename T, bool MUON>
__device__ __noinline__ void store_elements(const Args& a, const Tensor& t, T* p, int w, const float* x, int ld) {
  constexpr int U = 8;
  float rp[U];
  int at[U], in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) at[u] = -1;
  elements<U>(t, w, ld,
              [&](int u, int to, int from) {
                at[u] = to;
                in[u] = from;
                if (MUON) rp[u] = to_f(p[to]);
              },
              [&] {
#pragma unroll
                for (int u = 0; u < U; ++u)
                  if (at[u] >= 0) {
                    put(p + at[u], result<MUON>(a, t, x[in[u]], MUON ? rp[u] : 0.f));
                    at[u] = -1;
                  }
              });
}

// Columns [j0, j0 + w) (j0 a multiple of 8) into x, zeros up to the next multiple of 8 and in the rows that fill the
// tiles. `first`: the momentum buffer is still the old one.
template <int NT, typename T, bool MUON>
__device__ __forceinline__ void load_slice(const Args& a, const Tensor& t, long long base, int j0, int w, float* x,
                                           int ld, bool first) {
  const bool vec = vectors<T, MUON>(t, base, w);
  base += t.tall ? (long long)j0 * t.d : j0;
  const T* g = reinterpret_cast<const T*>(t.g) + base;
  float* m = MUON ? t.m + base : nullptr;
  if (vec && t.tall) {
    load_vectors<T, MUON, true>(a, t, g, m, w, x, ld, first);
  } else if (vec) {
    load_vectors<T, MUON, false>(a, t, g, m, w, x, ld, first);
  } else {
    load_elements<T, MUON>(a, t, g, m, w, x, ld, first);
  }
  const int w8 = (w + 7) & ~7;
  if (w < w8)
    for (int i = threadIdx.x >> 3; i < t.d; i += kThreads / 8) {
      const int j = (w8 - 8) + (threadIdx.x & 7);
      if (j >= w) x[i * ld + j] = 0.f;
    }
  if (t.d < NT * 8)
    for (int i = t.d; i < NT * 8; ++i)
      for (int j = threadIdx.x; j < w8; j += kThreads) x[i * ld + j] = 0.f;
}

template <typename T, bool MUON, bool TALL>
__device__ __forceinline__ void store_vectors(const Args& a, const Tensor& t, T* p, int w, float* x, int ld) {
  constexpr int N = Vec<T>::N, U = 4;
  const Walk<N> walk(a, t, w, ld);
  int at = walk.at;
  float* in = x + walk.in;
  for (int left = walk.n; left > 0; left -= U) {
    uint4 rp[U];
    if (MUON) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) rp[u] = *reinterpret_cast<const uint4*>(p + at + u * walk.step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < left) {
        Vec<T> v, was{};
        if (MUON) unpack(rp[u], was);
        move<false, N, TALL>(in + u * walk.in_step, ld, v.v);
#pragma unroll
        for (int k = 0; k < N; ++k) v.v[k] = result<MUON>(a, t, v.v[k], was.v[k]);
        *reinterpret_cast<uint4*>(p + at + u * walk.step) = repack(v);
      }
    }
    at += U * walk.step;
    in += U * walk.in_step;
  }
}

template <typename T, bool MUON>
__device__ __forceinline__ void store_slice(const Args& a, const Tensor& t, long long base, int j0, int w, float* x,
                                            int ld) {
  const bool vec = vectors<T, MUON>(t, base, w);
  base += t.tall ? (long long)j0 * t.d : j0;
  T* p = reinterpret_cast<T*>(t.p) + base;
  if (vec && t.tall) {
    store_vectors<T, MUON, true>(a, t, p, w, x, ld);
  } else if (vec) {
    store_vectors<T, MUON, false>(a, t, p, w, x, ld);
  } else {
    store_elements<T, MUON>(a, t, p, w, x, ld);
  }
}

// Tile (i, j), i <= j, of the packed upper triangle.
template <int NT>
__host__ __device__ constexpr int tri(int i, int j) {
  return i * NT - i * (i - 1) / 2 + j - i;
}

// Tile rows of a warp's tile group: all of them, or rows Q and 7 - Q of eight (nine tiles in every group).
template <int NT, int Q>
__host__ __device__ constexpr bool in_group(int i) {
  return Dims<NT>::GROUPS == 1 || i == Q || i == NT - 1 - Q;
}

// acc += the group's tiles of X X^T over columns 4 k .. 4 k + 3 for k = kg, kg + KG, ... The fragment of rows 8 i ..
// 8 i + 7 is the same as left and as right operand.
template <int NT, int Q>
__device__ __forceinline__ void gram(const float* x, int ld, int w, int kg, double (&acc)[Dims<NT>::ACC][2]) {
  const int lane = threadIdx.x & 31;
  const float* p = x + (lane >> 2) * ld + (lane & 3);
#pragma unroll (NT <= 2 ? 4 : 2)
  for (int k = kg * 4; k < w; k += Dims<NT>::KG * 4) {
    double f[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) f[i] = p[8 * i * ld + k];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (in_group<NT, Q>(i)) {
#pragma unroll
        for (int j = i; j < NT; ++j) dmma(acc[n++], f[i], f[j]);
      }
  }
}

// The group's tiles to or from (added) a packed upper triangle.
template <int NT, int Q, bool ADD>
__device__ __forceinline__ void pack(double* part, double (&acc)[Dims<NT>::ACC][2]) {
  const int lane = threadIdx.x & 31;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NT; ++i)
    if (in_group<NT, Q>(i)) {
#pragma unroll
      for (int j = i; j < NT; ++j, ++n) {
        double2* d = reinterpret_cast<double2*>(part + tri<NT>(i, j) * 64 + lane * 2);
        if (ADD) {
          acc[n][0] += d->x;
          acc[n][1] += d->y;
        } else {
          *d = make_double2(acc[n][0], acc[n][1]);
        }
      }
    }
}

template <int NT>
__device__ __forceinline__ void gram_group(int grp, const float* x, int ld, int w, int kg,
                                           double (&acc)[Dims<NT>::ACC][2]) {
  if constexpr (Dims<NT>::GROUPS == 1) {
    gram<NT, 0>(x, ld, w, kg, acc);
  } else {
    switch (grp) {
      case 0: gram<NT, 0>(x, ld, w, kg, acc); break;
      case 1: gram<NT, 1>(x, ld, w, kg, acc); break;
      case 2: gram<NT, 2>(x, ld, w, kg, acc); break;
      default: gram<NT, 3>(x, ld, w, kg, acc); break;
    }
  }
}
template <int NT, bool ADD>
__device__ __forceinline__ void pack_group(int grp, double* part, double (&acc)[Dims<NT>::ACC][2]) {
  if constexpr (Dims<NT>::GROUPS == 1) {
    pack<NT, 0, ADD>(part, acc);
  } else {
    switch (grp) {
      case 0: pack<NT, 0, ADD>(part, acc); break;
      case 1: pack<NT, 1, ADD>(part, acc); break;
      case 2: pack<NT, 2, ADD>(part, acc); break;
      default: pack<NT, 3, ADD>(part, acc); break;
    }
  }
}

// The warps' partial Gram matrices: halved until BUFS are left, then added in order. Calls f(q, sum q, sum q + 1) for the
// even q of the packed upper triangle. `work`: BUFS parts.
template <int NT, class F>
__device__ __forceinline__ void reduce_warps(double (&acc)[Dims<NT>::ACC][2], double* work, F&& f) {
  using D_ = Dims<NT>;
  const int warp = threadIdx.x >> 5, grp = warp % D_::GROUPS, kg = warp / D_::GROUPS;
#pragma unroll
  for (int h = D_::KG; h > D_::BUFS; h /= 2) {
    // the upper half goes through the buffers, as many at a time as there are
#pragma unroll
    for (int o = h / 2; o < h; o += D_::BUFS) {
      if (kg >= o && kg < o + D_::BUFS) pack_group<NT, false>(grp, work + (kg - o) * D_::PART, acc);
      __syncthreads();
      const int to = o - h / 2;
      if (kg >= to && kg < to + D_::BUFS && kg < h / 2) pack_group<NT, true>(grp, work + (kg - to) * D_::PART, acc);
      __syncthreads();
    }
  }
  if (kg < D_::BUFS) pack_group<NT, false>(grp, work + kg * D_::PART, acc);
  __syncthreads();
  for (int q = threadIdx.x * 2; q < D_::PART; q += kThreads * 2) {
    double2 s = *reinterpret_cast<const double2*>(work + q);
#pragma unroll
    for (int b = 1; b < D_::BUFS; ++b) {
      const double2 v = *reinterpret_cast<const double2*>(work + b * D_::PART + q);
      s.x += v.x;
      s.y += v.y;
    }
    f(q, s.x, s.y);
  }
}

// Tile n of the upper triangle.
template <int NT>
__device__ __forceinline__ void tile_of(int n, int& i, int& j) {
  i = 0;
#pragma unroll
  for (int k = 1; k < NT; ++k)
    if (n >= tri<NT>(k, k)) i = k;
  j = n - tri<NT>(i, i) + i;
}

// Element q of the packed upper triangle to both its places.
template <int NT>
__device__ __forceinline__ void spread(double* M, int q, double v) {
  int i, j;
  tile_of<NT>(q >> 6, i, j);
  M[(i * NT + j) * 64 + (q & 63)] = v;
  if (i != j) M[(j * NT + i) * 64 + (q & 7) * 8 + ((q >> 3) & 7)] = v;
}

// Places of an upper tile (i, j) in a matrix, for one lane: the rows of the left operand's tiles, of the right one's, the
// tile itself and its mirror image (offsets in doubles).
template <int NT>
struct Spot {
  int a, b, own, mirror;
  bool diagonal;
  __device__ __forceinline__ explicit Spot(int n) {
    int i, j;
    tile_of<NT>(n, i, j);
    set(i, j);
  }
  Spot() = default;
  __device__ __forceinline__ Spot(int i, int j) { set(i, j); }
  __device__ __forceinline__ void set(int i, int j) {
    const int lane = threadIdx.x & 31;
    a = i * NT * 64 + 2 * lane;
    b = j * NT * 64 + 2 * lane;
    own = (i * NT + j) * 64 + 2 * lane;
    mirror = (j * NT + i) * 64 + (lane & 3) * 16 + (lane >> 2);
    diagonal = i == j;
  }
};

// c = the tile of A B.
template <int NT>
__device__ __forceinline__ void product(const double* A, const double* B, const Spot<NT>& t, double (&c)[2]) {
  double2 a[NT], b[NT];
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    a[k] = *reinterpret_cast<const double2*>(A + t.a + 64 * k);
    b[k] = *reinterpret_cast<const double2*>(B + t.b + 64 * k);
  }
  double c1[2] = {0.0, 0.0};
  c[0] = c[1] = 0.0;
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    dmma(c, a[k].x, b[k].x);
    dmma(c1, a[k].y, b[k].y);
  }
  c[0] += c1[0];
  c[1] += c1[1];
}

// From 48 rows on PARTS warps take a tile row: its left operand stays in registers for the row's tiles (i, i + t), t up to
// half the tiles, columns wrapping around, which covers every pair once and gives each row as many. Calls f(place, c) for
// each tile of A B.
template <int NT, int PARTS, class F>
__device__ __forceinline__ void strip(const double2 (&a)[NT], const double* B, int i, int part, F&& f) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int t = part; t <= NT / 2; t += PARTS) {
    if (t == NT / 2 && i >= NT / 2) break;
    const int j = i + t < NT ? i + t : i + t - NT;
    const double* pb = B + j * NT * 64 + 2 * lane;
    double c[2] = {0.0, 0.0}, c1[2] = {0.0, 0.0};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const double2 b = *reinterpret_cast<const double2*>(pb + 64 * k);
      dmma(c, a[k].x, b.x);
      dmma(c1, a[k].y, b.y);
    }
    c[0] += c1[0];
    c[1] += c1[1];
    f(Spot<NT>(i, j), c);
  }
}
template <int NT>
__device__ __forceinline__ void load_row(const double* A, int i, double2 (&a)[NT]) {
#pragma unroll
  for (int k = 0; k < NT; ++k)
    a[k] = *reinterpret_cast<const double2*>(A + (i * NT + k) * 64 + 2 * (threadIdx.x & 31));
}

// Writes a tile and its mirror image. HALF: of a tile on the diagonal the upper half counts for both, as it must in G: S, a
// polynomial of G G^T, then is symmetric by itself, while an asymmetry that only G's diagonal tiles keep would grow by more
// than a^2 a step (eight steps on rank one: 3e-7 in the result, 6e-12 so).
template <int NT, bool HALF = false>
__device__ __forceinline__ void put_tile(double* M, const Spot<NT>& t, const double (&c)[2]) {
  if (!t.diagonal || !HALF) *reinterpret_cast<double2*>(M + t.own) = make_double2(c[0], c[1]);
  if (!t.diagonal) {
    M[t.mirror] = c[0];
    M[t.mirror + 8] = c[1];
  } else if (HALF) {
    const int lane = threadIdx.x & 31, r = lane >> 2, k = 2 * (lane & 3);
    if (r <= k) M[t.own] = M[t.mirror] = c[0];
    if (r <= k + 1) M[t.own + 1] = M[t.mirror + 8] = c[1];
  }
}

// c <- the tile of S = a I + b G + c G^2 from that of G^2.
template <int NT>
__device__ __forceinline__ void step_form(double (&c)[2], const double2& g, const Spot<NT>& t, double ca, double cb,
                                          double cc) {
  const int lane = threadIdx.x & 31, r = lane >> 2, k = 2 * (lane & 3);
  c[0] = cc * c[0] + (cb * g.x + (t.diagonal && r == k ? ca : 0.0));
  c[1] = cc * c[1] + (cb * g.y + (t.diagonal && r == k + 1 ? ca : 0.0));
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ void named_arrive(int id, int threads) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The steps for up to 16 rows, where latency is all. A warp has one of the NT x NT tiles, and no mirror image to write:
// the first half of the warps S, V and G' (the chain, which waits for itself alone), the second P', which follows with
// two S to take from. Named barriers: 1 the chain, 2 the P warps, 3 and 4 S is there (even and odd steps), 5 and 6 S has
// been read. At 16 x 16 a product on four warps, one to a matrix unit, takes 183 cycles with its barrier; on the three
// tiles of a triangle with their mirror images 212, and 310 where six warps share the units.
template <int NT>
__device__ __forceinline__ void iterate_small(const Args& a, double* G, double* work, double inv) {
  using D_ = Dims<NT>;
  constexpr int T = NT * NT;
  double *S = work, *V = work + 2 * D_::MAT, *M = work + 3 * D_::MAT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= 2 * T) return;
  const bool chain = warp < T;
  const int n = chain ? warp : warp - T;
  const Spot<NT> t(n / NT, n % NT);
  double c[2];
  if (chain) {
    double2 g = *reinterpret_cast<const double2*>(G + t.own);
    double sc = inv * inv;  // the first step's G still has to be scaled by it
    for (int step = 0;; ++step) {
      double* s = S + (step & 1) * D_::MAT;
      const double ca = a.coef[step][0], cb = a.coef[step][1] * sc, cc = a.coef[step][2] * sc * sc;
      product<NT>(G, G, t, c);
      step_form(c, g, t, ca, cb, cc);
      if (step >= 2) named_barrier(5 + (step & 1), 2 * T * 32);
      *reinterpret_cast<double2*>(s + t.own) = make_double2(c[0], c[1]);
      named_arrive(3 + (step & 1), 2 * T * 32);
      if (step + 1 == a.steps) return;
      named_barrier(1, T * 32);
      product<NT>(s, G, t, c);
      *reinterpret_cast<double2*>(V + t.own) = make_double2(c[0], c[1]);
      named_barrier(1, T * 32);
      product<NT>(s, V, t, c);
      g = make_double2(c[0] * sc, c[1] * sc);
      *reinterpret_cast<double2*>(G + t.own) = g;
      named_barrier(1, T * 32);
      sc = 1.0;
    }
  }
  for (int step = 0; step < a.steps; ++step) {
    const double* s = S + (step & 1) * D_::MAT;
    double *from = M + ((step + 1) & 1) * D_::MAT, *to = M + (step & 1) * D_::MAT;
    named_barrier(3 + (step & 1), 2 * T * 32);
    if (step) {
      product<NT>(s, from, t, c);
    } else {
      const double2 v = *reinterpret_cast<const double2*>(s + t.own);
      c[0] = v.x;
      c[1] = v.y;
    }
    *reinterpret_cast<double2*>(to + t.own) = make_double2(c[0], c[1]);
    if (step + 2 < a.steps) named_arrive(5 + (step & 1), 2 * T * 32);
    named_barrier(2, T * 32);
  }
}

// From the Gram matrix G of x (unscaled) to P with P x = the polynomial of x, in M[0] or M[1] (returned). work holds S (two
// up to 16 rows), V, M[0], M[1].
template <int NT, int WARPS>
__device__ double* iterate(const Args& a, double* G, double* work) {
  using D_ = Dims<NT>;
  double *S = work, *V = work + D_::MAT, *M = work + 2 * D_::MAT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double tr = 0.0;
  for (int i = NT <= 2 ? lane % D_::D : lane; i < D_::D; i += 32) tr += G[(i >> 3) * (NT + 1) * 64 + (i & 7) * 9];
#pragma unroll
  for (int o = NT == 1 ? 4 : NT == 2 ? 8 : 16; o; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o);
  const double inv = tr == 0.0 ? 0.0 : 1.0 / (sqrt(tr) + a.eps);  // zeros stay zeros however small eps is
  if constexpr (2 * NT * NT <= WARPS) {
    __syncthreads();  // every warp has its trace: the chain overwrites G without waiting for the others
    iterate_small<NT>(a, G, work, inv);
    M = work + 3 * D_::MAT;
  } else {
    // a warp's tiles: of S and of G' (R1 rounds), and of V and P' together (R2 rounds)
    constexpr int R1 = (D_::TILES + WARPS - 1) / WARPS, R2 = (2 * D_::TILES + WARPS - 1) / WARPS;
    Spot<NT> chain[R1], both[R2];
    if (NT < 6) {
#pragma unroll
      for (int q = 0; q < R1; ++q) chain[q] = Spot<NT>(min(warp + q * WARPS, D_::TILES - 1));
#pragma unroll
      for (int q = 0; q < R2; ++q) {
        const int n = warp + q * WARPS;
        both[q] = Spot<NT>(n < D_::TILES ? n : min(n - D_::TILES, D_::TILES - 1));
      }
    }
    double sc = inv * inv;  // the first step's G still has to be scaled by it
    for (int step = 0; step < a.steps; ++step) {
      const double ca = a.coef[step][0], cb = a.coef[step][1] * sc, cc = a.coef[step][2] * sc * sc;
      const bool last = step + 1 == a.steps;
      double *from = M + ((step + 1) & 1) * D_::MAT, *to = M + (step & 1) * D_::MAT;
      if constexpr (NT >= 6) {
        constexpr int PARTS = WARPS / NT;  // warps of a tile row
        const int line = warp % NT, part = warp / NT;
        double2 row[NT];
        if (part < PARTS) {
          load_row<NT>(G, line, row);
          strip<NT, PARTS>(row, G, line, part, [&](const Spot<NT>& t, double (&c)[2]) {
            const double2 g = *reinterpret_cast<const double2*>(G + t.own);
            step_form(c, g, t, ca, cb, cc);
            put_tile<NT>(S, t, c);
            if (step == 0) put_tile<NT>(to, t, c);
          });
        }
        __syncthreads();
        if (part < PARTS) {
          load_row<NT>(S, line, row);
          if (!last)
            strip<NT, PARTS>(row, G, line, part, [&](const Spot<NT>& t, double (&c)[2]) { put_tile<NT>(V, t, c); });
          if (step)
            strip<NT, PARTS>(row, from, line, part, [&](const Spot<NT>& t, double (&c)[2]) { put_tile<NT>(to, t, c); });
        }
        if (last) break;
        __syncthreads();
        if (part < PARTS)
          strip<NT, PARTS>(row, V, line, part, [&](const Spot<NT>& t, double (&c)[2]) {
            c[0] *= sc;
            c[1] *= sc;
            put_tile<NT, true>(G, t, c);
          });
      } else {
#pragma unroll
        for (int q = 0; q < R1; ++q) {
          if (warp + q * WARPS < D_::TILES) {
            const Spot<NT>& t = chain[q];
            const double2 g = *reinterpret_cast<const double2*>(G + t.own);
            double c[2];
            product<NT>(G, G, t, c);
            step_form(c, g, t, ca, cb, cc);
            put_tile<NT>(S, t, c);
            if (step == 0) put_tile<NT>(to, t, c);
          }
        }
        __syncthreads();
        // V = S G (but in the last step) and P' = S P (from the second on), each tile by its own warp
#pragma unroll
        for (int q = 0; q < R2; ++q) {
          const int n = warp + q * WARPS;
          const bool isv = n < D_::TILES;
          if (isv ? !last : n < 2 * D_::TILES && step > 0) {
            double c[2];
            product<NT>(S, isv ? G : from, both[q], c);
            put_tile<NT>(isv ? V : to, both[q], c);
          }
        }
        if (last) break;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < R1; ++q) {
          if (warp + q * WARPS < D_::TILES) {
            double c[2];
            product<NT>(S, V, chain[q], c);
            c[0] *= sc;
            c[1] *= sc;
            put_tile<NT, true>(G, chain[q], c);
          }
        }
      }
      __syncthreads();
      sc = 1.0;
    }
  }
  __syncthreads();
  double* P = M + ((a.steps - 1) & 1) * D_::MAT;
  for (int q = threadIdx.x; q < D_::MAT; q += WARPS * 32) P[q] *= inv;
  __syncthreads();
  return P;
}

// fp64 to fp32, to nearest. ODD: towards zero with the last bit set if anything was cut off, so that a later rounding to bf16
// (16 bits fewer) is the only one. What is cut off are the low 29 bits; below fp32's normal numbers it is more, and the bit is
// always set (a conversion back would tell, but the products took 6 to 8% longer with one).
template <bool ODD>
__device__ __forceinline__ float narrow(double v) {
  if constexpr (!ODD) return (float)v;
  const uint32_t f = __float_as_uint(__double2float_rz(v));
  const bool odd = (__double2loint(v) & 0x1fffffff) != 0 || (f & 0x7f800000u) == 0;
  return __uint_as_float(f | (odd ? 1u : 0u));
}
// Whether a result of type T goes through fp32 on its way to bf16. The Muon step's goes into an fp32 sum first.
template <typename T, bool MUON>
constexpr bool odd() {
  return !MUON && sizeof(T) == 2;
}

// x <- P x in place in fp64: a warp owns C groups of eight columns at a time. Up to 16 rows P stays in registers.
template <int NT, bool ODD>
__device__ __forceinline__ void apply(const double* P, float* x, int ld, int w) {
  constexpr int C = NT <= 4 ? 2 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const double2* p = reinterpret_cast<const double2*>(P) + lane;
  double2 held[NT <= 2 ? NT * NT : 1];
  if (NT <= 2) {
#pragma unroll
    for (int q = 0; q < NT * NT; ++q) held[q] = p[q * 32];
  }
  for (int j = warp * 8; j < w; j += kWarps * 8 * C) {
    double o[C][NT][2];
#pragma unroll
    for (int g = 0; g < C; ++g)
#pragma unroll
      for (int i = 0; i < NT; ++i) o[g][i][0] = o[g][i][1] = 0.0;
    const float* b = x + 2 * c * ld + j + r;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      double v[C][2];
#pragma unroll
      for (int g = 0; g < C; ++g) {
        const int at = j + g * kWarps * 8 < w ? g * kWarps * 8 : 0;  // a group past the end repeats the first
        v[g][0] = b[8 * k * ld + at];
        v[g][1] = b[(8 * k + 1) * ld + at];
      }
      double2 f[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) f[i] = NT <= 2 ? held[(i * NT + k) % (NT <= 2 ? NT * NT : 1)] : p[(i * NT + k) * 32];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < C; ++g) dmma(o[g][i], f[i].x, v[g][0]);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < C; ++g) dmma(o[g][i], f[i].y, v[g][1]);
    }
    __syncwarp();
#pragma unroll
    for (int g = 0; g < C; ++g)
      if (j + g * kWarps * 8 < w) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          *reinterpret_cast<float2*>(x + (8 * i + r) * ld + j + g * kWarps * 8 + 2 * c) =
              make_float2(narrow<ODD>(o[g][i][0]), narrow<ODD>(o[g][i][1]));
      }
  }
}

// The tensor that unit `at` (see Tensor::start) belongs to.
__device__ __forceinline__ const Tensor& tensor_of(const Args& a, long long at) {
  int ti = 0;
  for (int end = a.n; end - ti > 1;) {
    const int mid = (ti + end) / 2;
    if (a.t[mid].start <= at) ti = mid;
    else end = mid;
  }
  return a.t[ti];
}

// Resident: the blocks of a cluster hold one matrix, or a few short ones, `cap` columns each at most. Their parts of the
// Gram matrix go to every block of the matrix by asynchronous stores into its shared memory that the receiver's barrier
// counts: one way, and without the fence over the stores to the momentum buffer that a cluster barrier would need.
// Bound: one matrix at a time by latency (7.5 us for 12 matrices of 16 x 2048: of 13000 cycles 4100 the polynomial, 1650
// the last product, 1150 the loads); many by HBM and the fp64 units together (a Muon step of 1548 matrices of rank 16,
// 634 MB: 142 us, 4.5 TB/s, the units half busy; loads and stores alone take 106).
template <int NT, typename T, bool MUON>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 4 : 2) ortho_kernel(const __grid_constant__ Args a) {
  using D_ = Dims<NT>;
  extern __shared__ __align__(16) double sm[];
  __shared__ __align__(8) uint64_t bar;
  double *G = sm, *work = G + D_::MAT, *slots = work + D_::BUFS * D_::PART;
  float* x = reinterpret_cast<float*>(work + D_::work(a.blocks));
  const Tensor& t = tensor_of(a, blockIdx.x >> a.shift);
  // the blocks of this block's matrix: from `first` in the cluster, `rank` among them
  const int place = blockIdx.x & (a.blocks - 1), blocks = 1 << t.shift, rank = place & (blocks - 1), first = place - rank;
  const int ld = pitch(a.cap);
  if (a.blocks > 1) {
    if (threadIdx.x == 0 && blocks > 1) {
      mbar_init(&bar, 1);
      fence_mbar_init();
      mbar_arrive_expect_tx(&bar, (uint32_t)(blocks * D_::PART * sizeof(double)));
    }
    cluster_arrive();
  }
  const long long matrix = (((blockIdx.x >> a.shift) - t.start) << (a.shift - t.shift)) + (place >> t.shift);
  if (matrix >= t.batch) {  // the last cluster of a tensor is not full
    if (a.blocks > 1) {
      cluster_wait();
      cluster_arrive_relaxed();
      cluster_wait();
    }
    return;
  }
  const long long base = matrix * t.d * t.L;
  const int slice = (((t.L + blocks - 1) >> t.shift) + 7) & ~7;
  const int j0 = min(rank * slice, t.L), w = min(slice, t.L - j0);

  double acc[D_::ACC][2];
#pragma unroll
  for (int n = 0; n < D_::ACC; ++n) acc[n][0] = acc[n][1] = 0.0;
  if (w) load_slice<NT, T, MUON>(a, t, base, j0, w, x, ld, true);
  __syncthreads();
  gram<NT, 0>(x, ld, w, threadIdx.x >> 5, acc);
  if (a.blocks > 1) cluster_wait();  // every block's barrier is set up
  bool there = true;
  if (blocks > 1) {
    reduce_warps<NT>(acc, work, [&](int q, double v0, double v1) {
      for (int r = 0; r < blocks; ++r) push(slots + rank * D_::PART + q, &bar, first + r, v0, v1);
    });
    there = mbar_wait(&bar, 0, a.err, kDevErrWaitCluster, blockIdx.x);
    for (int q = threadIdx.x; q < D_::PART; q += kThreads) {
      double s = 0.0;
#pragma unroll 4
      for (int r = 0; r < blocks; ++r) s += slots[r * D_::PART + q];
      spread<NT>(G, q, s);
    }
  } else {
    reduce_warps<NT>(acc, work, [&](int q, double v0, double v1) {
      spread<NT>(G, q, v0);
      spread<NT>(G, q + 1, v1);
    });
  }
  if (a.blocks > 1) cluster_arrive_relaxed();  // for the exit: this block's pushes are under way
  // A part that did not come in time is recorded, and this block leaves its columns of the parameter or the output as they
  // were. The others' pushes may still be on their way into its shared memory: it stays until they have landed.
  if (!__syncthreads_and(there)) {
    cluster_wait();
    mbar_wait(&bar, 0, a.err, kDevErrWaitCluster, blockIdx.x);
    return;
  }
  const double* P = iterate<NT, kWarps>(a, G, work);
  apply<NT, odd<T, MUON>()>(P, x, ld, w);
  __syncthreads();
  if (w) store_slice<T, MUON>(a, t, base, j0, w, x, ld);
  if (a.blocks > 1) cluster_wait();
}

// Split: block b of a matrix takes the chunks b, b + blocks, ... of `cap` columns. Bound by the fp64 units: 192 x 64 x 2048
// in 82 us, 49 at their rate (here and below a kernel alone with cold caches; a pass of the three takes 277); three blocks to
// an SM where the registers allow it, as two (94 us) leave the units idle while a block loads.
template <int NT, typename T, bool MUON>
__global__ void __launch_bounds__(kThreads, NT == 6 || MUON || sizeof(T) == 2 ? 2 : 3)
    gram_kernel(const __grid_constant__ Args a) {
  using D_ = Dims<NT>;
  extern __shared__ __align__(16) double sm[];
  double* work = sm;
  float* x = reinterpret_cast<float*>(work + D_::BUFS * D_::PART);
  const int block = blockIdx.x % a.blocks, ld = pitch(a.cap), warp = threadIdx.x >> 5;
  const long long mat = a.first + blockIdx.x / a.blocks;
  const Tensor& t = tensor_of(a, mat);
  const long long base = (mat - t.start) * t.d * t.L;
  double acc[D_::ACC][2];
#pragma unroll
  for (int n = 0; n < D_::ACC; ++n) acc[n][0] = acc[n][1] = 0.0;
  for (int j0 = block * a.cap; j0 < t.L; j0 += a.blocks * a.cap) {
    const int w = min(a.cap, t.L - j0);
    load_slice<NT, T, MUON>(a, t, base, j0, w, x, ld, true);
    __syncthreads();
    gram_group<NT>(warp % D_::GROUPS, x, ld, w, warp / D_::GROUPS, acc);
    __syncthreads();
  }
  double* part = a.gram + (long long)blockIdx.x * D_::PART;
  reduce_warps<NT>(acc, work, [&](int q, double v0, double v1) {
    *reinterpret_cast<double2*>(part + q) = make_double2(v0, v1);
  });
}

template <int NT>
constexpr int form_warps() {
  return NT >= 6 ? 16 : kWarps;
}

// One block per matrix: the parts in order, then P. 192 matrices of 64 rows: 76 us, two rounds on 148 SMs at 55% of the fp64
// units (104 us with a tile of a product at a time on eight warps).
template <int NT>
__global__ void __launch_bounds__(form_warps<NT>() * 32) form_kernel(const __grid_constant__ Args a) {
  using D_ = Dims<NT>;
  constexpr int FT = form_warps<NT>() * 32;
  extern __shared__ __align__(16) double sm[];
  double *G = sm, *work = G + D_::MAT;
  const double* part = a.gram + (long long)blockIdx.x * a.blocks * D_::PART;
  for (int q = threadIdx.x * 2; q < D_::PART; q += FT * 2) {
    double2 s = make_double2(0.0, 0.0);
#pragma unroll 8
    for (int b = 0; b < a.blocks; ++b) {
      const double2 v = *reinterpret_cast<const double2*>(part + (long long)b * D_::PART + q);
      s.x += v.x;
      s.y += v.y;
    }
    spread<NT>(G, q, s.x);
    spread<NT>(G, q + 1, s.y);
  }
  __syncthreads();
  const double* P = iterate<NT, form_warps<NT>()>(a, G, work);
  double* out = a.form + (long long)blockIdx.x * D_::MAT;
  for (int q = threadIdx.x; q < D_::MAT; q += FT) out[q] = P[q];
}

// Split: x <- P x, read and written once more. Bound by the fp64 units (192 x 64 x 2048: 133 us, 87 at their
// rate); as many blocks to an SM as the registers of the load allow.
template <int NT, typename T, bool MUON>
__global__ void __launch_bounds__(kThreads, NT >= 6 && !MUON && sizeof(T) == 4 ? 3 : 2)
    product_kernel(const __grid_constant__ Args a) {
  using D_ = Dims<NT>;
  extern __shared__ __align__(16) double sm[];
  float* x = reinterpret_cast<float*>(sm + D_::MAT);
  const int block = blockIdx.x % a.blocks, ld = pitch(a.cap);
  const long long mat = blockIdx.x / a.blocks;
  const Tensor& t = tensor_of(a, a.first + mat);
  const long long base = (a.first + mat - t.start) * t.d * t.L;
  const double* form = a.form + mat * D_::MAT;
  for (int q = threadIdx.x; q < D_::MAT; q += kThreads) sm[q] = form[q];
  for (int j0 = block * a.cap; j0 < t.L; j0 += a.blocks * a.cap) {
    const int w = min(a.cap, t.L - j0);
    load_slice<NT, T, MUON>(a, t, base, j0, w, x, ld, false);
    __syncthreads();
    apply<NT, odd<T, MUON>()>(sm, x, ld, w);
    __syncthreads();
    store_slice<T, MUON>(a, t, base, j0, w, x, ld);
    __syncthreads();
  }
}

// An unevaluated sum of two doubles, about 106 bits: Knuth's two-sum and the exact product by fma (intrinsics, which the
// compiler does not contract).
struct Pair {
  double h, l;
};
__device__ __forceinline__ Pair two_sum(double a, double b) {
  const double s = __dadd_rn(a, b), v = __dsub_rn(s, a);
  return {s, __dadd_rn(__dsub_rn(a, __dsub_rn(s, v)), __dsub_rn(b, v))};
}
// c += a b, the low parts of the sum unnormalised.
__device__ __forceinline__ void add_product(Pair& c, const Pair& a, const Pair& b) {
  const double p = __dmul_rn(a.h, b.h);
  const double e = __fma_rn(a.l, b.h, __fma_rn(a.h, b.l, __fma_rn(a.h, b.h, -p)));
  const Pair s = two_sum(c.h, p);
  c.h = s.h;
  c.l = __dadd_rn(c.l, __dadd_rn(s.l, e));
}
// The same with an exact x (an fp32 value).
__device__ __forceinline__ void add_product(Pair& c, const Pair& a, double x) {
  const double p = __dmul_rn(a.h, x);
  const Pair s = two_sum(c.h, p);
  c.h = s.h;
  c.l = __dadd_rn(c.l, __dadd_rn(s.l, __fma_rn(a.l, x, __fma_rn(a.h, x, -p))));
}
// c += p, exact.
__device__ __forceinline__ void add(Pair& c, double p) {
  const Pair s = two_sum(c.h, p);
  c.h = s.h;
  c.l = __dadd_rn(c.l, s.l);
}
__device__ __forceinline__ Pair times(const Pair& a, const Pair& b) {
  Pair c{0.0, 0.0};
  add_product(c, a, b);
  return two_sum(c.h, c.l);
}

// A symmetric d x d matrix of pairs in shared memory, rows of an odd pitch.
struct Wide {
  double *h, *l;
  int ld;
  __device__ __forceinline__ Pair at(int i, int j) const { return {h[i * ld + j], l[i * ld + j]}; }
  __device__ __forceinline__ void put(int i, int j, const Pair& v) const {
    h[i * ld + j] = h[j * ld + i] = v.h;
    l[i * ld + j] = l[j * ld + i] = v.l;
  }
};

constexpr int kMaxPairs = kMaxD * (kMaxD + 1) / 2, kPairRounds = (kMaxPairs + kThreads - 1) / kThreads;

// Columns [j0, j0 + w) into x [d][ld] element by element, in the order of memory.
template <typename T, bool MUON>
__device__ __forceinline__ void load_columns(const Args& a, const Tensor& t, long long base, int j0, int w, float* x, int ld,
                                             bool first) {
  for (int e = threadIdx.x; e < w * t.d; e += kThreads) {
    const int c = t.tall ? e / t.d : e % w, i = t.tall ? e % t.d : e / w;
    const long long at = base + (t.tall ? (long long)j0 * t.d + e : (long long)i * t.L + j0 + c);
    float v = to_f(reinterpret_cast<const T*>(t.g)[at]);
    if (MUON) {
      float m = t.m[at];
      v = update(a, v, m, first);
      if (first) t.m[at] = m;
    }
    x[i * ld + c] = v;
  }
}

// One block for one matrix, all of it in pairs of doubles: the Gram matrix (products of fp32 values are exact in fp64), the
// steps, and P x, for which x is read a second time. A thread has up to nine elements of the upper triangle, or with few
// rows a share of the columns of one. Bound by the fp64 units of the SM that has the matrix (a product and its sum take 8 to
// 14 of their instructions, where the kernels above take one on the matrix units): 16 steps on 12 matrices of 16 x 2048
// 0.37 ms, on 1548 of 16 x 1024 1.4, on 192 of 64 x 2048 8.7, on one of 64 x 40000 47. Polynomials this long are rare, so
// the columns of a matrix are not spread over more blocks.
template <typename T, bool MUON>
__global__ void __launch_bounds__(kThreads) careful_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) double sm[];
  const Tensor& t = tensor_of(a, blockIdx.x);
  const long long base = ((long long)blockIdx.x - t.start) * t.d * t.L;
  const int tid = threadIdx.x, d = t.d, pd = d | 1, count = d * (d + 1) / 2, ld = a.cap + 1;
  const Wide G{sm, sm + d * pd, pd}, S{sm + 2 * d * pd, sm + 3 * d * pd, pd}, P{sm + 4 * d * pd, sm + 5 * d * pd, pd};
  uint16_t* place = reinterpret_cast<uint16_t*>(sm + 6 * d * pd);  // (row, column) of each element of the upper triangle
  float* x = reinterpret_cast<float*>(place + ((count + 7) & ~7));
  for (int q = tid; q < d * d; q += kThreads) {
    const int i = q / d, j = q - i * d;
    if (j >= i) place[i * d - i * (i - 1) / 2 + j - i] = (uint16_t)(i << 8 | j);
  }
  const int groups = max(kThreads / count, 1), group = groups > 1 ? tid / count : 0;
  Pair r[kPairRounds];
#pragma unroll
  for (int q = 0; q < kPairRounds; ++q) r[q] = {0.0, 0.0};
  // calls f(element, its row, its column, r[q]) for the thread's elements
  auto each = [&](auto&& f) {
#pragma unroll
    for (int q = 0; q < kPairRounds; ++q)
      if (tid + q * kThreads < count) {
        const int at = place[tid + q * kThreads];
        f(at >> 8, at & 255, r[q]);
      }
  };
  auto product = [&](const Wide& A, const Wide& B) {
    each([&](int i, int j, Pair& c) {
      c = {0.0, 0.0};
      for (int k = 0; k < d; ++k) add_product(c, A.at(i, k), B.at(j, k));
      c = two_sum(c.h, c.l);
    });
  };
  auto write = [&](const Wide& M) {
    each([&](int i, int j, const Pair& c) { M.put(i, j, c); });
  };

  for (int j0 = 0; j0 < t.L; j0 += a.cap) {
    const int w = min(a.cap, t.L - j0);
    load_columns<T, MUON>(a, t, base, j0, w, x, ld, true);
    __syncthreads();
    auto dot = [&](int i, int j, int c0, int step, Pair& s) {
      for (int c = c0; c < w; c += step) add(s, __dmul_rn((double)x[i * ld + c], (double)x[j * ld + c]));
    };
    if (groups > 1) {
      if (group < groups) {
        const int at = place[tid - group * count];
        dot(at >> 8, at & 255, group, groups, r[0]);
      }
    } else {
      each([&](int i, int j, Pair& s) { dot(i, j, 0, 1, s); });
    }
    __syncthreads();
  }
  if (groups > 1) {
    Pair* share = reinterpret_cast<Pair*>(x);
    share[tid] = r[0];
    __syncthreads();
    if (tid < count)
      for (int g = 1; g < groups; ++g) {
        const Pair o = share[g * count + tid], s = two_sum(r[0].h, o.h);
        r[0] = {s.h, r[0].l + (s.l + o.l)};
      }
  }
  each([&](int i, int j, Pair& c) {
    c = two_sum(c.h, c.l);
    G.put(i, j, c);
  });
  __syncthreads();
  double tr = 0.0;
  for (int i = 0; i < d; ++i) tr += G.h[i * pd + i];
  const double inv = tr == 0.0 ? 0.0 : 1.0 / (sqrt(tr) + a.eps), sq = __dmul_rn(inv, inv);
  const Pair scale{sq, __fma_rn(inv, inv, -sq)};
  __syncthreads();
  each([&](int i, int j, Pair& c) { G.put(i, j, times(c, scale)); });
  __syncthreads();
  for (int step = 0; step < a.steps; ++step) {
    const double ca = a.coef[step][0], cb = a.coef[step][1], cc = a.coef[step][2];
    product(G, G);
    each([&](int i, int j, const Pair& c) {  // S = a I + b G + c G^2
      Pair s{i == j ? ca : 0.0, 0.0};
      add_product(s, G.at(i, j), {cb, 0.0});
      add_product(s, c, {cc, 0.0});
      s = two_sum(s.h, s.l);
      S.put(i, j, s);
      if (step == 0) P.put(i, j, s);
    });
    __syncthreads();
    if (step) {
      product(S, P);
      __syncthreads();
      write(P);
    }
    if (step + 1 == a.steps) break;
    product(S, G);
    __syncthreads();
    write(G);  // S G
    __syncthreads();
    product(S, G);
    __syncthreads();
    write(G);  // S G S
    __syncthreads();
  }
  __syncthreads();

  for (int j0 = 0; j0 < t.L; j0 += a.cap) {
    const int w = min(a.cap, t.L - j0);
    load_columns<T, MUON>(a, t, base, j0, w, x, ld, false);
    __syncthreads();
    for (int e = tid; e < w * d; e += kThreads) {
      const int c = t.tall ? e / d : e % w, i = t.tall ? e % d : e / w;
      Pair o{0.0, 0.0};
      for (int k = 0; k < d; ++k) add_product(o, P.at(i, k), (double)x[k * ld + c]);
      T* p = reinterpret_cast<T*>(t.p) + base + (t.tall ? (long long)j0 * d + e : (long long)i * t.L + j0 + c);
      put(p, result<MUON>(a, t, narrow<odd<T, MUON>()>((o.h + o.l) * inv), MUON ? to_f(*p) : 0.f));
    }
    __syncthreads();
  }
}

// Factor of a division of a number below 2^16 by n > 1: the high word of the product is the quotient.
uint32_t by(int n) { return (uint32_t)((1ull << 32) / n + 1); }

void set_cap(Args& a, int cap) {
  a.cap = cap;
  for (int k = 0; k < 2; ++k) {
    const int vectors = cap / (k ? 8 : 4);
    a.rows[k] = kThreads / vectors;
    a.by_v[k] = by(vectors);
    a.by_rows[k] = by(a.rows[k]);
  }
}

// Raises the kernel's limit of shared memory on this device, never lowers it: another thread may be about to launch it with
// the size that it has asked for.
template <auto KERN>
int raise_smem(long long bytes) {
  static std::mutex mu;
  static std::atomic<long long> raised[64];
  int dev = 0;
  SMELB_CUDA(cudaGetDevice(&dev));
  SMELB_CHECK_ARG(dev < 64, kErrArg, "orthogonalize: device %d", dev);
  if (raised[dev].load(std::memory_order_acquire) >= bytes) return kOk;
  std::lock_guard<std::mutex> lk(mu);
  if (raised[dev].load(std::memory_order_relaxed) < bytes) {
    SMELB_CUDA(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    raised[dev].store(bytes, std::memory_order_release);
  }
  return kOk;
}

template <auto KERN>
int launch(const Args& a, long long blocks, int threads, long long smem, int cluster, cudaStream_t st) {
  SMELB_CHECK_ARG(blocks < (1LL << 31), kErrShape, "orthogonalize: %lld blocks", blocks);
  if (int rc = raise_smem<KERN>(smem)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  SMELB_CUDA(cudaLaunchKernelEx(&cfg, KERN, a));
  count_launch();
  return kOk;
}

// Columns of a resident block at most: 47 KB for 16 rows (four blocks to an SM; 1024 columns in two ran 7% slower on 1548
// matrices of 16 x 512 .. 2048), 106 KB for 32 (two blocks in clusters of up to four).
constexpr int kMaxBlocks = 8;
constexpr int kBlockCols = 512;

// Whether matrices of this size are held by a cluster: up to 32 rows, and no more columns than eight blocks hold (1548
// matrices of rank 16 the split way: 225 us a step against 142; 512 x 16 x 2048: 80 against 64).
bool resident(int nt, int L) { return nt <= 4 && L <= kBlockCols * kMaxBlocks; }

// Blocks that a resident matrix needs.
int blocks_needed(int L) {
  int c = 1;
  while (L > kBlockCols * c) c *= 2;
  return c;
}

static_assert(sizeof(Args) <= 4096, "kernel parameters");

// Matrices of one round of the split way: their partial Gram matrices and P are the workspace (50 KB each at 64 rows).
constexpr long long kSplitRound = 4096;

// Blocks for one matrix of the split way: as many chunks to each as leave eight blocks for an SM, and at most 296 for one
// matrix (their partial Gram matrices are added by one block).
int split_blocks(int nt, long long matrices, int L) {
  const long long chunks = (L + split_cap(nt) - 1) / split_cap(nt);
  const long long per =
      std::max({1LL, chunks * std::min(matrices, kSplitRound) / (148 * 8), (chunks + 295) / 296});
  return (int)((chunks + per - 1) / per);
}

int log2_of(int c) { return c == 8 ? 3 : c / 2; }

template <int NT, typename T, bool MUON>
int run_resident(Args& a, long long matrices, int maxL, cudaStream_t st) {
  using D_ = Dims<NT>;
  // few matrices: more blocks for each, down to 256 columns, until two are on every SM, and the same for all. Many: each
  // as many as it needs, short ones side by side in a cluster (a short matrix spread over the blocks of a long one would
  // form P in each of them, and a launch of its own would leave SMs idle at its end: 1548 matrices in 191, 154 and, as
  // here, 142 us).
  int c = blocks_needed(maxL);
  const bool few = matrices * c <= 148 * 4;
  while (few && c < kMaxBlocks && maxL > 256 * c && matrices * c < 296) c *= 2;
  a.blocks = c;
  a.shift = log2_of(c);
  long long clusters = 0;
  int cap = 32;
  for (int k = 0; k < a.n; ++k) {
    Tensor& t = a.t[k];
    t.shift = few ? a.shift : log2_of(blocks_needed(t.L));
    t.start = clusters;
    clusters += (t.batch + (c >> t.shift) - 1) >> (a.shift - t.shift);
    cap = std::max(cap, (((t.L + (1 << t.shift) - 1) >> t.shift) + 31) / 32 * 32);
  }
  set_cap(a, cap);
  const long long smem = (long long)(D_::MAT + D_::work(c)) * 8 + (long long)NT * 8 * pitch(a.cap) * 4;
  return launch<ortho_kernel<NT, T, MUON>>(a, clusters * c, kThreads, smem, c, st);
}

template <int NT, typename T, bool MUON>
int run_split(Args& a, long long matrices, int maxL, double* ws, cudaStream_t st) {
  using D_ = Dims<NT>;
  a.blocks = split_blocks(NT, matrices, maxL);
  set_cap(a, split_cap(NT));
  const long long x = (long long)NT * 8 * pitch(a.cap) * 4;
  const int blocks = a.blocks;
  for (a.first = 0; a.first < matrices; a.first += kSplitRound) {
    const long long n = std::min(kSplitRound, matrices - a.first);
    a.gram = ws;
    a.form = ws + n * blocks * D_::PART;
    if (int rc = launch<gram_kernel<NT, T, MUON>>(a, n * blocks, kThreads, (long long)D_::BUFS * D_::PART * 8 + x, 1, st))
      return rc;
    if (int rc = launch<form_kernel<NT>>(a, n, form_warps<NT>() * 32, (long long)(D_::MAT + D_::POLY) * 8, 1, st))
      return rc;
    if (int rc = launch<product_kernel<NT, T, MUON>>(a, n * blocks, kThreads, (long long)D_::MAT * 8 + x, 1, st))
      return rc;
  }
  return kOk;
}

// How much the rounding of G grows until the last step reads it, at most.
double growth(int steps, const double* coef) {
  double g = 1.0, most = 1.0;
  for (int s = 0; s + 1 < steps; ++s) {
    g = std::max(g, 1.0) * coef[3 * s] * coef[3 * s];
    most = g > most || g != g ? g : most;
  }
  return most;
}
// Up to here 0.45 * 2^-53 * 2^26 is a twentieth of a rounding to fp32.
constexpr double kMaxGrowth = 67108864.0;

template <typename T, bool MUON>
int run_careful(Args& a, int nt, long long matrices, cudaStream_t st) {
  const int d = nt * 8;
  a.cap = std::min(512, kMaxD * kMaxD / d / 32 * 32);
  const long long x = std::max((long long)d * (a.cap + 1) * 4, (long long)kThreads * 16);
  const long long smem = 6LL * d * (d | 1) * 8 + (d * (d + 1) / 2 + 7) / 8 * 16 + x;
  return launch<careful_kernel<T, MUON>>(a, matrices, kThreads, smem, 1, st);
}

template <int NT, typename T, bool MUON>
int run_way(Args& a, long long matrices, int maxL, bool held, double* ws, cudaStream_t st) {
  if constexpr (NT <= 4)
    if (held) return run_resident<NT, T, MUON>(a, matrices, maxL, st);
  return run_split<NT, T, MUON>(a, matrices, maxL, ws, st);
}

template <int NT>
int run_typed(Args& a, bool bf, bool muon, long long matrices, int maxL, bool held, double* ws, cudaStream_t st) {
  if (muon)
    return bf ? run_way<NT, bf16, true>(a, matrices, maxL, held, ws, st)
              : run_way<NT, float, true>(a, matrices, maxL, held, ws, st);
  return bf ? run_way<NT, bf16, false>(a, matrices, maxL, held, ws, st)
            : run_way<NT, float, false>(a, matrices, maxL, held, ws, st);
}

// Row tiles that the kernels are built for.
int tiles_for(int d) {
  const int n = (d + 7) / 8;
  return n <= 4 ? n : n <= 6 ? 6 : 8;
}
constexpr int kTileCounts[] = {1, 2, 3, 4, 6, 8};

int check_shapes(const smelb_muon_tensor* t, int64_t n, const char* what) {
  SMELB_CHECK_ARG(t || n == 0, kErrArg, "%s: null pointer", what);
  for (int64_t i = 0; i < n; ++i) {
    SMELB_CHECK_ARG(t[i].batch >= 0 && t[i].rows >= 1 && t[i].cols >= 1 && std::min(t[i].rows, t[i].cols) <= kMaxD &&
                        std::max(t[i].rows, t[i].cols) < (1LL << 24) && t[i].batch < (1LL << 28),
                    kErrShape, "%s: tensor %lld: %lld x %lld x %lld (short side 1..%d)", what, (long long)i,
                    (long long)t[i].batch, (long long)t[i].rows, (long long)t[i].cols, kMaxD);
  }
  return kOk;
}

// Calls f(row tiles, held, the launch's tensors idx[0 .. count), matrices, longest side) for every launch: tensors of the
// same row tiles and way, at most kMaxTensors.
template <typename F>
int for_launches(const smelb_muon_tensor* t, int64_t n, F&& f) {
  for (int nt : kTileCounts)
    for (int held = 0; held < 2; ++held) {
      int64_t idx[kMaxTensors];
      int count = 0, maxL = 0;
      long long matrices = 0;
      for (int64_t i = 0; i < n; ++i) {
        const int d = (int)std::min(t[i].rows, t[i].cols), L = (int)std::max(t[i].rows, t[i].cols);
        if (t[i].batch == 0 || tiles_for(d) != nt || resident(nt, L) != (held != 0)) continue;
        idx[count++] = i;
        matrices += t[i].batch;
        maxL = std::max(maxL, L);
        if (count == kMaxTensors) {
          if (int rc = f(nt, held != 0, idx, count, matrices, maxL)) return rc;
          count = maxL = 0;
          matrices = 0;
        }
      }
      if (count)
        if (int rc = f(nt, held != 0, idx, count, matrices, maxL)) return rc;
    }
  return kOk;
}

// Bytes that the split launches of a call need, the largest of them (a launch reuses the one before's).
long long workspace(const smelb_muon_tensor* t, int64_t n) {
  long long most = 0;
  for_launches(t, n, [&](int nt, bool held, const int64_t*, int, long long matrices, int maxL) {
    if (!held) {
      const long long part = nt * (nt + 1) / 2 * 64, form = nt * nt * 64;
      most = std::max(most, std::min(matrices, kSplitRound) * (split_blocks(nt, matrices, maxL) * part + form) * 8);
    }
    return 0;
  });
  return most;
}

// Refuses tensors of which one that is written shares memory with another (out of an orthogonalisation may be x itself).
int check_overlap(const smelb_muon_tensor* t, int64_t n, int bytes, bool muon, const char* what) {
  struct Span {
    uintptr_t lo, hi;
    int64_t tensor;
    bool written;
  };
  std::unique_ptr<Span[]> spans(new (std::nothrow) Span[(size_t)n * 3]);
  SMELB_CHECK_ARG(spans || n == 0, kErrArg, "%s: no host memory for %lld tensors", what, (long long)n);
  int64_t count = 0;
  for (int64_t i = 0; i < n; ++i) {
    const uintptr_t e = (uintptr_t)(t[i].batch * t[i].rows * t[i].cols);
    auto span = [&](const void* at, int size, bool written) {
      if (e) spans[count++] = {(uintptr_t)at, (uintptr_t)at + e * size, i, written};
    };
    span(t[i].p, bytes, true);
    if (muon || t[i].g != t[i].p) span(t[i].g, bytes, false);
    if (muon) span(t[i].m, 4, true);
  }
  std::sort(spans.get(), spans.get() + count, [](const Span& a, const Span& b) { return a.lo < b.lo; });
  const Span *any = nullptr, *out = nullptr;  // those that reach farthest so far, of all and of the written ones
  for (const Span* s = spans.get(); s < spans.get() + count; ++s) {
    const Span* hit = s->written ? any : out;
    SMELB_CHECK_ARG(!hit || hit->hi <= s->lo, kErrArg, "%s: tensors %lld and %lld share memory that is written", what,
                    (long long)hit->tensor, (long long)s->tensor);
    if (!any || s->hi > any->hi) any = s;
    if (s->written && (!out || s->hi > out->hi)) out = s;
  }
  return kOk;
}

int run(const smelb_muon_tensor* t, int64_t n, int dtype, bool muon, double lr, double mu, bool nesterov, double wd,
        int adjust, int steps, const double* coef, double eps, void* ws, int64_t ws_bytes, const char* what,
        cudaStream_t st) {
  if (int rc = check_shapes(t, n, what)) return rc;
  for (int64_t i = 0; i < n; ++i)
    SMELB_CHECK_ARG(t[i].batch == 0 || (t[i].p && t[i].g && (t[i].m || !muon)), kErrArg, "%s: null pointer", what);
  SMELB_CHECK_ARG(dtype == 0 || dtype == 1, kErrDtype, "%s: dtype %d", what, dtype);
  SMELB_CHECK_ARG(steps >= 1 && steps <= kMaxSteps && coef, kErrArg, "%s: %d steps (1..%d)", what, steps, kMaxSteps);
  SMELB_CHECK_ARG(eps > 0.0, kErrArg, "%s: eps must be positive", what);
  if (int rc = check_overlap(t, n, dtype == 1 ? 2 : 4, muon, what)) return rc;
  const long long need = workspace(t, n);
  SMELB_CHECK_ARG(ws_bytes >= need && (ws || !need), kErrWorkspace, "%s: workspace %lld bytes, %lld needed", what,
                  (long long)ws_bytes, need);
  SMELB_CHECK_ARG(((uintptr_t)ws & 255) == 0, kErrArg, "%s: workspace must be 256-byte aligned", what);
  bool any = false;
  for (int64_t i = 0; i < n; ++i) any = any || t[i].batch > 0;
  if (!any) return kOk;
  int dev = 0;
  SMELB_CUDA(cudaGetDevice(&dev));
  Args a{};
  a.err = device_status_on(dev, st);
  a.steps = steps;
  a.mu = (float)mu;
  a.omu = (float)(1.0 - mu);
  a.nesterov = nesterov;
  a.decay = (float)(1.0 - lr * wd);
  a.eps = eps;
  for (int s = 0; s < steps; ++s)
    for (int k = 0; k < 3; ++k) a.coef[s][k] = coef[3 * s + k];
  const bool careful = !(growth(steps, coef) <= kMaxGrowth);
  return for_launches(t, n, [&](int nt, bool held, const int64_t* idx, int count, long long matrices, int maxL) {
    a.n = count;
    long long start = 0;
    for (int k = 0; k < count; ++k) {
      const smelb_muon_tensor& s = t[idx[k]];
      const int d = (int)std::min(s.rows, s.cols), L = (int)std::max(s.rows, s.cols);
      const double f = adjust == 1 ? 0.2 * sqrt((double)L) : sqrt(std::max(1.0, (double)s.rows / (double)s.cols));
      // a single column is a single row in memory
      a.t[k] = Tensor{s.p, s.g, s.m, start, (int)s.batch, 0, d, L, s.rows > s.cols && d > 1 ? 1 : 0, by(d),
                      {by(kThreads * 4 / d), by(kThreads * 8 / d)}, (float)(lr * f)};
      start += s.batch;
    }
    const bool bf = dtype == 1;
    if (careful) {
      if (muon) return bf ? run_careful<bf16, true>(a, nt, matrices, st) : run_careful<float, true>(a, nt, matrices, st);
      return bf ? run_careful<bf16, false>(a, nt, matrices, st) : run_careful<float, false>(a, nt, matrices, st);
    }
    double* w = (double*)ws;
    switch (nt) {
      case 1: return run_typed<1>(a, bf, muon, matrices, maxL, held, w, st);
      case 2: return run_typed<2>(a, bf, muon, matrices, maxL, held, w, st);
      case 3: return run_typed<3>(a, bf, muon, matrices, maxL, held, w, st);
      case 4: return run_typed<4>(a, bf, muon, matrices, maxL, held, w, st);
      case 6: return run_typed<6>(a, bf, muon, matrices, maxL, held, w, st);
      default: return run_typed<8>(a, bf, muon, matrices, maxL, held, w, st);
    }
  });
}

}  // namespace
}  // namespace smelb

using namespace smelb;

extern "C" {

int64_t smelb_muon_workspace_bytes(const smelb_muon_tensor* tensors, int64_t n) {
  if (n < 0 || check_shapes(tensors, n, "muon_workspace_bytes") != kOk) return -1;
  return workspace(tensors, n);
}

int64_t smelb_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
  const smelb_muon_tensor t{nullptr, nullptr, nullptr, batch, rows, cols};
  return smelb_muon_workspace_bytes(&t, 1);
}

int smelb_orthogonalize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
                        const double* coefficients, double eps, void* out, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  const smelb_muon_tensor t{out, x, nullptr, batch, rows, cols};
  return run(&t, 1, dtype, false, 0.0, 0.0, false, 0.0, 0, steps, coefficients, eps, workspace, workspace_bytes,
             "orthogonalize", (cudaStream_t)stream);
}

int smelb_muon_step(const smelb_muon_tensor* tensors, int64_t n, int dtype, double lr, double momentum, int nesterov,
                    double weight_decay, int adjust, int steps, const double* coefficients, double eps, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  SMELB_CHECK_ARG(n >= 0 && (adjust == 0 || adjust == 1), kErrArg, "muon_step: n=%lld adjust=%d", (long long)n, adjust);
  return run(tensors, n, dtype, true, lr, momentum, nesterov != 0, weight_decay, adjust, steps, coefficients, eps,
             workspace, workspace_bytes, "muon_step", (cudaStream_t)stream);
}

}  // extern "C"

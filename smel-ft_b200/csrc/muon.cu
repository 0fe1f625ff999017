// Orthogonalised updates of LoRA factors: x -> the Newton-Schulz polynomial of x, alone or inside a momentum step.
//
//   X0 = x / (|x|_F + eps);   X <- a X + b (X X^T) X + c (X X^T)^2 X,  `steps` times, on the short side d <= 64.
//
// Every iterate is a polynomial in G0 = X0 X0^T times X0, so the long side is needed only twice: once for the Gram
// matrix and once for the product P X0. Between them, on d x d matrices that commute and are symmetric:
//   S = a I + b G + c G^2;   P <- S P;   G <- S G S.
// Precision. The steps grow a singular value near zero by a^steps (485 for the usual polynomial), and an error delta in
// G moves the result by delta / sigma^2, so gradients of low rank (few tokens reached the expert) come out up to 3e-4
// off when G is held in fp32. G and the d x d matrices are fp64, on the fp64 matrix instruction (m8n8k4): at d = 16
// that is 4 operations per byte of x, below the card's 5.7 (37 TFLOP/s over 6.4 TB/s), so it costs no time on long
// factors.
//
// One cluster of 1, 2, 4 or 8 blocks per matrix. A block keeps its slice of the long side in shared memory as fp32
// [d][columns] whatever the layout in memory (a slice that does not fit is read a second time); partial Gram matrices
// are added over the cluster in rank order through distributed shared memory, and each block forms P for itself.
#include <algorithm>

#include "common.cuh"
#include "host.h"
#include "smelb.h"

namespace smelb {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kMaxSteps = 16, kMaxTensors = 64, kMaxD = 64;

struct Tensor {
  void* p;        // parameter (momentum step) or output
  const void* g;  // gradient or input
  float* m;       // momentum buffer
  long long start;  // matrices before this tensor's
  int d, L;       // short and long side
  int tall;       // memory is [L][d] (else [d][L])
  float step;     // lr * shape factor
};

struct Args {
  Tensor t[kMaxTensors];
  int n, steps, cluster, cap;  // cap: columns that a block holds at once
  float mu, omu, decay;  // omu: 1 - momentum, from 64 bits
  int nesterov;
  double eps;
  double coef[kMaxSteps][3];
};

template <int NT>
struct Dims {
  static constexpr int D = NT * 8, LDM = D + 4;            // row pitch of the fp64 matrices: conflict-free fragments
  static constexpr int TILES = NT * (NT + 1) / 2;          // tiles of the upper triangle
  static constexpr int GROUPS = NT == 8 ? 4 : 1;           // tile groups among the warps (accumulators in registers)
  static constexpr int KG = kWarps / GROUPS;               // warps that split the columns
  static constexpr int BUFS = KG < 4 ? KG : 4;             // partial Gram matrices in shared memory at once
  static constexpr int MAT = D * LDM;                      // doubles of one matrix
  static constexpr int PART = TILES * 64;                  // doubles of one packed upper triangle
  // G, S, P, V, then this block's part of the Gram matrix; the warps' partial sums alias S, P and V
  static constexpr int WORK = (3 * MAT > BUFS * PART ? 3 * MAT : BUFS * PART);
  static constexpr long long kFixed = (long long)(MAT + WORK + PART) * 8;
};

// Column pitch 8 mod 32 and columns of rows 4-7 (mod 8) shifted by four: the fragments of the Gram product (8 rows x 4
// columns) and of the product with P (4 rows x 8 columns) then both touch 32 different banks.
__device__ __forceinline__ int xat(int i, int j, int ld) { return i * ld + (j ^ (i & 4)); }

__device__ __forceinline__ void dmma(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
               : "+d"(c[0]), "+d"(c[1])
               : "d"(a), "d"(b));
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ double ld_cluster(const double* p, int rank) {
  uint32_t a;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a));
  return v;
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// One element of the input: the gradient, or the momentum update, whose new buffer is written when `first`.
template <typename T, bool MUON>
__device__ __forceinline__ float element(const Args& a, const Tensor& t, long long at, bool first) {
  const float g = to_f(reinterpret_cast<const T*>(t.g)[at]);
  if (!MUON) return g;
  float m = t.m[at];
  if (first) {
    m = fmaf(a.mu, m, a.omu * g);
    t.m[at] = m;
  }
  return a.nesterov ? fmaf(a.mu, m, a.omu * g) : m;
}

// Columns [j0, j0 + w) into x, zeros up to the next multiple of 8.
template <typename T, bool MUON>
__device__ void load_slice(const Args& a, const Tensor& t, long long base, int j0, int w, float* x, int ld, int D,
                           bool first) {
  if (t.tall) {
    for (int q = threadIdx.x; q < w * t.d; q += kThreads) {
      const int j = q / t.d, i = q - j * t.d;
      x[xat(i, j, ld)] = element<T, MUON>(a, t, base + (long long)j0 * t.d + q, first);
    }
  } else {
    for (int i = 0; i < t.d; ++i)
      for (int j = threadIdx.x; j < w; j += kThreads)
        x[xat(i, j, ld)] = element<T, MUON>(a, t, base + (long long)i * t.L + j0 + j, first);
  }
  const int w8 = (w + 7) & ~7;
  for (int i = threadIdx.x >> 3; i < t.d; i += kThreads / 8) {
    const int j = (w8 - 8) + (threadIdx.x & 7);
    if (j >= w) x[xat(i, j, ld)] = 0.f;
  }
  for (int q = threadIdx.x; q < (D - t.d) * w8; q += kThreads) x[xat(t.d + q / w8, q % w8, ld)] = 0.f;
}

template <typename T, bool MUON>
__device__ __forceinline__ void emit(const Args& a, const Tensor& t, long long at, float o) {
  T* p = reinterpret_cast<T*>(t.p) + at;
  put(p, MUON ? fmaf(-t.step, o, to_f(*p) * a.decay) : o);
}

template <typename T, bool MUON>
__device__ void store_slice(const Args& a, const Tensor& t, long long base, int j0, int w, const float* x, int ld) {
  if (t.tall) {
    for (int q = threadIdx.x; q < w * t.d; q += kThreads) {
      const int j = q / t.d, i = q - j * t.d;
      emit<T, MUON>(a, t, base + (long long)j0 * t.d + q, x[xat(i, j, ld)]);
    }
  } else {
    for (int i = 0; i < t.d; ++i)
      for (int j = threadIdx.x; j < w; j += kThreads)
        emit<T, MUON>(a, t, base + (long long)i * t.L + j0 + j, x[xat(i, j, ld)]);
  }
}

// Tile rows of a warp's tile group: all of them, or rows Q and 7 - Q of eight (nine tiles in every group).
template <int NT, int Q>
__host__ __device__ constexpr bool in_group(int i) {
  return Dims<NT>::GROUPS == 1 || i == Q || i == NT - 1 - Q;
}

// acc += the group's tiles of X X^T over columns 4 k .. 4 k + 3 for k = kg, kg + KG, ... The fragment of rows 8 i ..
// 8 i + 7 is the same as left and as right operand.
template <int NT, int Q>
__device__ __forceinline__ void gram(const float* x, int ld, int w, int kg, double (&acc)[Dims<NT>::TILES][2]) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  for (int k = kg * 4; k < w; k += Dims<NT>::KG * 4) {
    double f[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) f[i] = x[xat(8 * i + r, k + c, ld)];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = i; j < NT; ++j, ++n)
        if (in_group<NT, Q>(i)) dmma(acc[n], f[i], f[j]);
  }
}

// Adds or writes the group's tiles into a packed upper triangle.
template <int NT, int Q, bool ADD>
__device__ __forceinline__ void pack(double* part, double (&acc)[Dims<NT>::TILES][2]) {
  const int lane = threadIdx.x & 31;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = i; j < NT; ++j, ++n)
      if (in_group<NT, Q>(i)) {
        double* d = part + n * 64 + lane * 2;
        if (ADD) {
          acc[n][0] += d[0];
          acc[n][1] += d[1];
        } else {
          d[0] = acc[n][0];
          d[1] = acc[n][1];
        }
      }
}

// c = rows 8 i .. of A times columns 8 j .. of B, both symmetric.
template <int NT>
__device__ __forceinline__ void product(const double* A, const double* B, int i, int j, double (&c)[2]) {
  constexpr int LDM = Dims<NT>::LDM;
  const int lane = threadIdx.x & 31;
  const double* pa = A + (8 * i + (lane >> 2)) * LDM + (lane & 3);
  const double* pb = B + (8 * j + (lane >> 2)) * LDM + (lane & 3);
  c[0] = c[1] = 0.0;
#pragma unroll
  for (int k = 0; k < NT * 2; ++k) dmma(c, pa[4 * k], pb[4 * k]);
}

// Writes a tile and its mirror image.
template <int NT>
__device__ __forceinline__ void put_tile(double* M, int i, int j, const double (&c)[2]) {
  constexpr int LDM = Dims<NT>::LDM;
  const int lane = threadIdx.x & 31, r = 8 * i + (lane >> 2), k = 8 * j + 2 * (lane & 3);
  M[r * LDM + k] = c[0];
  M[r * LDM + k + 1] = c[1];
  if (i != j) {
    M[k * LDM + r] = c[0];
    M[(k + 1) * LDM + r] = c[1];
  }
}

// Tile n of the upper triangle.
template <int NT>
__device__ __forceinline__ void tile_of(int n, int& i, int& j) {
  i = 0;
  while (n >= NT - i) n -= NT - i++;
  j = i + n;
}

// From the Gram matrix G (unscaled) to P with P x = the polynomial of x; leaves P in M[2].
template <int NT>
__device__ void iterate(const Args& a, double* G, double* S, double* P, double* V) {
  using D_ = Dims<NT>;
  constexpr int LDM = D_::LDM, PER = (D_::TILES + kWarps - 1) / kWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double tr = 0.0;
  for (int i = 0; i < D_::D; ++i) tr += G[i * LDM + i];
  const double inv = 1.0 / (sqrt(tr) + a.eps);
  double sc = inv * inv;  // the first step's G still has to be scaled by it
  for (int step = 0; step < a.steps; ++step) {
    const double ca = a.coef[step][0], cb = a.coef[step][1] * sc, cc = a.coef[step][2] * sc * sc;
    const bool last = step + 1 == a.steps;
    for (int n = warp; n < D_::TILES; n += kWarps) {
      int i, j;
      tile_of<NT>(n, i, j);
      double c[2];
      product<NT>(G, G, i, j, c);
      const int r = 8 * i + (lane >> 2), k = 8 * j + 2 * (lane & 3);
      c[0] = cb * G[r * LDM + k] + cc * c[0] + (r == k ? ca : 0.0);
      c[1] = cb * G[r * LDM + k + 1] + cc * c[1] + (r == k + 1 ? ca : 0.0);
      put_tile<NT>(S, i, j, c);
      if (step == 0) put_tile<NT>(P, i, j, c);
    }
    __syncthreads();
    double np[PER][2], nv[PER][2];
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int n = warp + q * kWarps;
      if (n < D_::TILES) {
        int i, j;
        tile_of<NT>(n, i, j);
        if (step) product<NT>(S, P, i, j, np[q]);
        if (!last) product<NT>(S, G, i, j, nv[q]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int n = warp + q * kWarps;
      if (n < D_::TILES) {
        int i, j;
        tile_of<NT>(n, i, j);
        if (step) put_tile<NT>(P, i, j, np[q]);
        if (!last) put_tile<NT>(V, i, j, nv[q]);
      }
    }
    __syncthreads();
    if (!last) {
      for (int n = warp; n < D_::TILES; n += kWarps) {
        int i, j;
        tile_of<NT>(n, i, j);
        double c[2];
        product<NT>(S, V, i, j, c);
        c[0] *= sc;
        c[1] *= sc;
        put_tile<NT>(G, i, j, c);
      }
      __syncthreads();
    }
    sc = 1.0;
  }
  for (int i = threadIdx.x; i < D_::D * D_::D; i += kThreads) P[(i / D_::D) * LDM + i % D_::D] *= inv;
  __syncthreads();
}

// x <- P x in place: a warp owns eight columns at a time.
template <int NT>
__device__ void apply(const double* P, float* x, int ld, int w) {
  constexpr int LDM = Dims<NT>::LDM;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  for (int j = warp * 8; j < w; j += kWarps * 8) {
    double b[NT * 2];
#pragma unroll
    for (int k = 0; k < NT * 2; ++k) b[k] = x[xat(4 * k + c, j + r, ld)];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      double o[2] = {0.0, 0.0};
#pragma unroll
      for (int k = 0; k < NT * 2; ++k) dmma(o, P[(8 * i + r) * LDM + 4 * k + c], b[k]);
      *reinterpret_cast<float2*>(x + xat(8 * i + r, j + 2 * c, ld)) = make_float2((float)o[0], (float)o[1]);
    }
  }
}

template <int NT, typename T, bool MUON>
__global__ void __launch_bounds__(kThreads) ortho_kernel(const __grid_constant__ Args a) {
  using D_ = Dims<NT>;
  extern __shared__ __align__(16) double sm[];
  double *G = sm, *work = sm + D_::MAT, *part = work + D_::WORK;
  double *S = work, *P = work + D_::MAT, *V = work + 2 * D_::MAT;
  float* x = reinterpret_cast<float*>(part + D_::PART);
  const int warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % a.cluster, ld = a.cap + 8;
  const long long mat = blockIdx.x / a.cluster;
  int ti = 0;
  while (ti + 1 < a.n && a.t[ti + 1].start <= mat) ++ti;
  const Tensor& t = a.t[ti];
  const long long base = (mat - t.start) * (long long)t.d * t.L;
  const int slice = ((t.L + a.cluster - 1) / a.cluster + 7) & ~7;
  const int s0 = min(rank * slice, t.L), s1 = min(s0 + slice, t.L);
  const int chunks = (s1 - s0 + a.cap - 1) / a.cap;

  const int grp = warp % D_::GROUPS, kg = warp / D_::GROUPS;
  double acc[D_::TILES][2];
#pragma unroll
  for (int n = 0; n < D_::TILES; ++n) acc[n][0] = acc[n][1] = 0.0;
  for (int ch = 0; ch < chunks; ++ch) {
    const int j0 = s0 + ch * a.cap, w = min(a.cap, s1 - j0);
    if (ch) __syncthreads();
    load_slice<T, MUON>(a, t, base, j0, w, x, ld, D_::D, true);
    __syncthreads();
    switch (grp) {
      case 0: gram<NT, 0>(x, ld, w, kg, acc); break;
      case 1: gram<NT, 1>(x, ld, w, kg, acc); break;
      case 2: gram<NT, 2>(x, ld, w, kg, acc); break;
      default: gram<NT, 3>(x, ld, w, kg, acc); break;
    }
  }
  // the warps' partial sums, halved until BUFS are left, then added in order
  auto pack_group = [&](double* dst, bool add) {
    switch (grp) {
      case 0: add ? pack<NT, 0, true>(dst, acc) : pack<NT, 0, false>(dst, acc); break;
      case 1: add ? pack<NT, 1, true>(dst, acc) : pack<NT, 1, false>(dst, acc); break;
      case 2: add ? pack<NT, 2, true>(dst, acc) : pack<NT, 2, false>(dst, acc); break;
      default: add ? pack<NT, 3, true>(dst, acc) : pack<NT, 3, false>(dst, acc); break;
    }
  };
#pragma unroll
  for (int h = D_::KG; h > D_::BUFS; h /= 2) {
    if (kg >= h / 2 && kg < h) pack_group(work + (kg - h / 2) * D_::PART, false);
    __syncthreads();
    if (kg < h / 2) pack_group(work + kg * D_::PART, true);
    __syncthreads();
  }
  if (kg < D_::BUFS) pack_group(work + kg * D_::PART, false);
  __syncthreads();
  for (int q = threadIdx.x; q < D_::PART; q += kThreads) {
    double s = work[q];
#pragma unroll
    for (int b = 1; b < D_::BUFS; ++b) s += work[b * D_::PART + q];
    part[q] = s;
  }
  if (a.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int q = threadIdx.x; q < D_::PART; q += kThreads) {
    double s = 0.0;
    if (a.cluster > 1)
      for (int r = 0; r < a.cluster; ++r) s += ld_cluster(part + q, r);
    else
      s = part[q];
    int i, j;
    tile_of<NT>(q >> 6, i, j);
    const int r = 8 * i + ((q & 63) >> 3), k = 8 * j + (q & 7);
    G[r * D_::LDM + k] = s;
    if (i != j) G[k * D_::LDM + r] = s;
  }
  if (a.cluster > 1) cluster_arrive();  // this block has read the others' parts
  __syncthreads();
  iterate<NT>(a, G, S, P, V);
  for (int ch = chunks - 1; ch >= 0; --ch) {  // the last chunk is still there
    const int j0 = s0 + ch * a.cap, w = min(a.cap, s1 - j0);
    if (ch < chunks - 1) {
      __syncthreads();
      load_slice<T, MUON>(a, t, base, j0, w, x, ld, D_::D, false);
      __syncthreads();
    }
    apply<NT>(P, x, ld, w);
    __syncthreads();
    store_slice<T, MUON>(a, t, base, j0, w, x, ld);
  }
  if (a.cluster > 1) cluster_wait();  // its part stays until every block has read it
}

constexpr int kSmemMax = 227 * 1024;

// Columns of x that a block of NT row tiles can hold.
template <int NT>
constexpr int max_cols() {
  return (int)((kSmemMax - Dims<NT>::kFixed) / (NT * 8 * 4) - 8) / 32 * 32;
}

template <int NT, typename T, bool MUON>
int launch(Args& a, long long matrices, int maxL, cudaStream_t st) {
  int c = 1;
  while (c < 8 && maxL > 256 * c) c *= 2;
  const int slice = ((maxL + c - 1) / c + 31) / 32 * 32;
  a.cluster = c;
  a.cap = std::min(slice, max_cols<NT>());
  const long long smem = Dims<NT>::kFixed + (long long)NT * 8 * (a.cap + 8) * 4;
  SMELB_CHECK_ARG(matrices * c < (1LL << 31), kErrShape, "orthogonalize: %lld matrices", matrices);
  auto kern = ortho_kernel<NT, T, MUON>;
  SMELB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(matrices * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)c, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  SMELB_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  count_launch();
  return kOk;
}

template <int NT>
int launch_typed(Args& a, bool bf, bool muon, long long matrices, int maxL, cudaStream_t st) {
  if (muon) return bf ? launch<NT, bf16, true>(a, matrices, maxL, st) : launch<NT, float, true>(a, matrices, maxL, st);
  return bf ? launch<NT, bf16, false>(a, matrices, maxL, st) : launch<NT, float, false>(a, matrices, maxL, st);
}

// Row tiles that the kernel is built for.
int tiles_for(int d) {
  const int n = (d + 7) / 8;
  return n <= 4 ? n : n <= 6 ? 6 : 8;
}

int run(const smelb_muon_tensor* t, int64_t n, int dtype, bool muon, double lr, double mu, bool nesterov, double wd,
        int adjust, int steps, const double* coef, double eps, const char* what, cudaStream_t st) {
  SMELB_CHECK_ARG(t || n == 0, kErrArg, "%s: null pointer", what);
  SMELB_CHECK_ARG(dtype == 0 || dtype == 1, kErrDtype, "%s: dtype %d", what, dtype);
  SMELB_CHECK_ARG(steps >= 1 && steps <= kMaxSteps && coef, kErrArg, "%s: %d steps (1..%d)", what, steps, kMaxSteps);
  SMELB_CHECK_ARG(eps > 0.0, kErrArg, "%s: eps must be positive", what);
  for (int64_t i = 0; i < n; ++i) {
    SMELB_CHECK_ARG(t[i].batch >= 0 && t[i].rows >= 1 && t[i].cols >= 1 && std::min(t[i].rows, t[i].cols) <= kMaxD &&
                        std::max(t[i].rows, t[i].cols) < (1LL << 24) && t[i].batch < (1LL << 31),
                    kErrShape, "%s: tensor %lld: %lld x %lld x %lld (short side 1..%d)", what, (long long)i,
                    (long long)t[i].batch, (long long)t[i].rows, (long long)t[i].cols, kMaxD);
    SMELB_CHECK_ARG(t[i].batch == 0 || (t[i].p && t[i].g && (t[i].m || !muon)), kErrArg, "%s: null pointer", what);
  }
  Args a{};
  a.steps = steps;
  a.mu = (float)mu;
  a.omu = (float)(1.0 - mu);
  a.nesterov = nesterov;
  a.decay = (float)(1.0 - lr * wd);
  a.eps = eps;
  for (int s = 0; s < steps; ++s)
    for (int k = 0; k < 3; ++k) a.coef[s][k] = coef[3 * s + k];
  for (int nt : {1, 2, 3, 4, 6, 8}) {
    long long matrices = 0;
    int maxL = 0;
    a.n = 0;
    auto flush = [&]() -> int {
      if (!a.n) return kOk;
      const bool bf = dtype == 1;
      const int rc = nt == 1   ? launch_typed<1>(a, bf, muon, matrices, maxL, st)
                     : nt == 2 ? launch_typed<2>(a, bf, muon, matrices, maxL, st)
                     : nt == 3 ? launch_typed<3>(a, bf, muon, matrices, maxL, st)
                     : nt == 4 ? launch_typed<4>(a, bf, muon, matrices, maxL, st)
                     : nt == 6 ? launch_typed<6>(a, bf, muon, matrices, maxL, st)
                               : launch_typed<8>(a, bf, muon, matrices, maxL, st);
      a.n = 0;
      matrices = 0;
      maxL = 0;
      return rc;
    };
    for (int64_t i = 0; i < n; ++i) {
      const int d = (int)std::min(t[i].rows, t[i].cols), L = (int)std::max(t[i].rows, t[i].cols);
      if (t[i].batch == 0 || tiles_for(d) != nt) continue;
      const double ratio = (double)t[i].rows / (double)t[i].cols;
      const double f = adjust == 1 ? 0.2 * sqrt((double)L) : sqrt(std::max(1.0, ratio));
      a.t[a.n++] = Tensor{t[i].p, t[i].g, t[i].m, matrices, d, L, t[i].rows > t[i].cols ? 1 : 0, (float)(lr * f)};
      matrices += t[i].batch;
      maxL = std::max(maxL, L);
      if (a.n == kMaxTensors)
        if (int rc = flush()) return rc;
    }
    if (int rc = flush()) return rc;
  }
  return kOk;
}

}  // namespace
}  // namespace smelb

using namespace smelb;

extern "C" {

int smelb_orthogonalize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
                        const double* coefficients, double eps, void* out, void* stream) {
  const smelb_muon_tensor t{out, x, nullptr, batch, rows, cols};
  return run(&t, 1, dtype, false, 0.0, 0.0, false, 0.0, 0, steps, coefficients, eps, "orthogonalize",
             (cudaStream_t)stream);
}

int smelb_muon_step(const smelb_muon_tensor* tensors, int64_t n, int dtype, double lr, double momentum, int nesterov,
                    double weight_decay, int adjust, int steps, const double* coefficients, double eps, void* stream) {
  SMELB_CHECK_ARG(n >= 0 && (adjust == 0 || adjust == 1), kErrArg, "muon_step: n=%lld adjust=%d", (long long)n, adjust);
  return run(tensors, n, dtype, true, lr, momentum, nesterov != 0, weight_decay, adjust, steps, coefficients, eps,
             "muon_step", (cudaStream_t)stream);
}

}  // extern "C"

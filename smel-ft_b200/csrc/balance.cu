// The router's balance loss with its gradient, and per-expert usage statistics: reductions of the routing tables
// probs [T, E] and topi [T, K] over the tokens, per sequence of a packed batch.
//
//   n_s     rows of sequence s that the mask keeps
//   c[s,e]  their choices of expert e;  P[s,e] = sum of their probs[., e]
//   loss    = 1/S' sum_s (E / (K n_s^2)) sum_e c[s,e] P[s,e]     over the S' sequences with n_s > 0
//   d loss / d probs[t,e] = (E c[s,e] / (K n_s^2)) / S' on the kept rows of s, 0 on every other row
//
// Two launches forward: one block per tile of rows sums the tile's rows of each sequence it meets into a record, then
// one block per (sequence, 32 experts) adds a sequence's records in order. Nothing is added in an order that depends
// on timing (integer counts aside, where it does not matter), so equal inputs give equal bits. A tile b and a
// sequence s that meet have the record b + s: going down the rows either the tile or the sequence advances by one, so
// the sums are distinct and T / rows + S records are enough for any lengths.
// Sums: fp32 within a tile (at most kMaxTileRows rows), fp64 across tiles.
//
// Bound: HBM for long tables, latency for a micro-batch. On a B200: tiles of 131072 x 256 in 37 us (3.7 TB/s), of 4096 x 256
// in 5; the finishing launch 6 to 10 us; the gradient of 131072 x 256 in 23 us (5.8 TB/s written).
#include <algorithm>

#include "common.cuh"
#include "host.h"
#include "smelb.h"

namespace smelb {
namespace {

constexpr int kTileThreads = 512;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kMaxTileRows = 128;
constexpr int kMaxE = 512, kMaxK = 32;
// A finishing block adds COLS experts of one sequence with kFinThreads / COLS threads each: 32 where sequences are many, 8
// where the records of few of them are long lists (one sequence of 65537 rows and 128 experts, 586 records: 16 us in four
// blocks of 32 experts).
constexpr int kFinThreads = 512;

struct TileArgs {
  const float* probs;
  long long ld;
  const long long* topi;
  const void* topv;  // usage only
  int topv_f32;
  const uint8_t* mask;
  const int* cu;
  int S, E, K, rows;
  uint32_t by_k;  // 2^32 / K + 1 (K > 1)
  long long T;
  float* rec_mass;    // [records][E]
  float* rec_weight;  // [records][E], usage only
  int* rec_cnt;       // [records][E]
  int* rec_n;         // [records]
  int* ticket;        // zeroed here for the finalising launch
  int* err;
};

// Rows [lo, hi) of sequence s, clamped into [0, T] (all rows without cu_seqlens).
__device__ __forceinline__ void seq_range(const int* cu, int s, long long T, long long& lo, long long& hi) {
  lo = 0;
  hi = T;
  if (cu) {
    lo = min((long long)max(cu[s], 0), T);
    hi = min((long long)max(cu[s + 1], 0), T);
  }
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// The sequences that can hold rows t0 .. t1: those from the first that ends behind t0 to the first that ends behind t1
// (counted by the whole block, in one pass over their ends).
__device__ __forceinline__ void sequences_of(const int* cu, int S, long long t0, long long t1, int& s0, int& s1) {
  s0 = s1 = 0;
  if (cu)
    for (int base = 0; base < S; base += blockDim.x) {
      const int s = base + threadIdx.x;
      const long long end = s < S ? cu[s + 1] : t1 + 1;
      s0 += __syncthreads_count(end <= t0);
      s1 += __syncthreads_count(end <= t1);
    }
}

// The sequence that holds row t (-1: none), among s0 .. s1.
__device__ __forceinline__ int sequence_of(const int* cu, int S, long long t, int s0, int s1) {
  if (!cu) return 0;
  while (s0 < s1) {
    const int mid = (s0 + s1) >> 1;
    if (cu[mid + 1] <= t) s0 = mid + 1;
    else s1 = mid;
  }
  return s0 < S && cu[s0] <= t && t < cu[s0 + 1] ? s0 : -1;
}

// A tile's rows by runs of one sequence. A run of kWarpRows rows or more, or a tile's only one, is summed by the block;
// shorter ones, of which a tile of short sequences has many, by a warp each (a run costs the block 1.5 us of barriers).
constexpr int kWarpRows = 32;
struct Runs {
  int seq[kMaxTileRows];         // sequence of each row
  int begin[kMaxTileRows + 1];   // first row of each run, then the number of rows
  int in_warp[kMaxTileRows / 32];
  int n;
};
__device__ __forceinline__ void find_runs(Runs& runs, const int* cu, int S, long long t0, int rows) {
  const int tid = threadIdx.x, lane = tid & 31;
  int s0, s1;
  sequences_of(cu, S, t0, t0 + rows - 1, s0, s1);
  if (s0 == s1 && s0 < S && cu[s0] <= t0) {  // as most tiles of long sequences: one run
    if (tid == 0) {
      runs.seq[0] = s0;
      runs.begin[0] = 0;
      runs.begin[1] = rows;
      runs.n = 1;
    }
    __syncthreads();
    return;
  }
  if (tid < rows) runs.seq[tid] = sequence_of(cu, S, t0 + tid, s0, s1);
  __syncthreads();
  const bool head = tid < rows && (tid == 0 || runs.seq[tid] != runs.seq[tid - 1]);
  const unsigned heads = __ballot_sync(0xffffffffu, head);
  if (lane == 0 && tid < kMaxTileRows) runs.in_warp[tid / 32] = __popc(heads);
  __syncthreads();
  if (tid < kMaxTileRows) {
    int k = __popc(heads & ((1u << lane) - 1));
    for (int w = 0; w < tid / 32; ++w) k += runs.in_warp[w];
    if (head) runs.begin[k] = tid;
    if (tid == kMaxTileRows - 1) {
      runs.n = k + (head ? 1 : 0);
      runs.begin[runs.n] = rows;
    }
  }
  __syncthreads();
}

// One run by one warp: rows [ra, rb), less than kWarpRows of them. h: the warp's table of counts.
template <int VEC>
__device__ __forceinline__ void warp_run(const TileArgs& a, const uint8_t* ok, int* h, long long t0, int ra, int rb,
                                         long long rec) {
  const int lane = threadIdx.x & 31, E = a.E, K = a.K;
  for (int e = lane; e < E; e += 32) h[e] = 0;
  __syncwarp();  // the lanes add to each other's entries, and a vote orders no memory
  const bool mine = ra + lane < rb && ok[ra + lane];
  const unsigned kept = __ballot_sync(0xffffffffu, mine);
  for (int i = ra * K + lane; i < rb * K; i += 32)
    if (ok[K == 1 ? i : (int)__umulhi((uint32_t)i, a.by_k)]) {
      const long long v = a.topi[t0 * K + i];
      if (v >= 0 && v < E) atomicAdd(&h[(int)v], 1);
      else dev_fail(a.err, kDevErrBadIndex);
    }
  __syncwarp();
  for (int col = lane * VEC; col < E; col += 32 * VEC) {
    const float* p = a.probs + t0 * a.ld + col;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
#pragma unroll 4
    for (int r = ra; r < rb; ++r) {
      float v[VEC];
      if constexpr (VEC == 4) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p + r * a.ld));
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
      } else {
        v[0] = __ldg(p + r * a.ld);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += (kept >> (r - ra)) & 1 ? v[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) a.rec_mass[rec * E + col + j] = acc[j];
  }
  for (int e = lane; e < E; e += 32) a.rec_cnt[rec * E + e] = h[e];
  if (lane == 0) a.rec_n[rec] = __popc(kept);
  __syncwarp();
}

// KIND: the loss over one sequence, the loss over packed ones, or the usage statistics (one sequence). Blocks to an SM by
// what their registers hold without spilling in the loops (packed: 74 us a pass of 131072 x 256 at two, 86 at three).
enum TileKind { kOne, kPacked, kUsage };
template <int VEC, int KIND>
__global__ void __launch_bounds__(kTileThreads, KIND == kUsage ? 4 : KIND == kPacked ? 2 : 3)
    balance_tile_kernel(const TileArgs a) {
  constexpr bool USAGE = KIND == kUsage, PACKED = KIND == kPacked;
  __shared__ uint8_t ok[kMaxTileRows];
  __shared__ int cnt[kMaxE];
  __shared__ float red[kTileThreads * VEC];
  __shared__ Runs runs;  // packed
  extern __shared__ float hist[];  // [kTileWarps][E]: the warps' weights (usage), or counts (short sequences)
  const int tid = threadIdx.x, E = a.E, K = a.K;
  const long long t0 = (long long)blockIdx.x * a.rows;
  const int rows = (int)min((long long)a.rows, a.T - t0);
  // the tile's rows are on their way to L2 while the block finds out which of them count
  if (a.ld == E) {
    const char* p = reinterpret_cast<const char*>(a.probs + t0 * E);
    for (int b = tid * 128; b < rows * E * 4; b += kTileThreads * 128) prefetch_l2(p + b);
  }
  for (int b = tid * 128; b < rows * K * 8; b += kTileThreads * 128)
    prefetch_l2(reinterpret_cast<const char*>(a.topi + t0 * K) + b);
  if (blockIdx.x == 0 && tid == 0) *a.ticket = 0;
  if (tid < rows) ok[tid] = a.mask ? a.mask[t0 + tid] != 0 : 1;
  const int ncol = (E + VEC - 1) / VEC, lanes = kTileThreads / ncol;
  const int lane = tid / ncol, col = (tid - lane * ncol) * VEC;
  int n_runs = 1;
  if constexpr (PACKED) {
    find_runs(runs, a.cu, a.S, t0, rows);
    n_runs = runs.n;
    if (n_runs > 1)
      for (int k = tid >> 5; k < n_runs; k += kTileWarps) {
        const int ra = runs.begin[k], rb = runs.begin[k + 1], s = runs.seq[ra];
        if (s >= 0 && rb - ra < kWarpRows)
          warp_run<VEC>(a, ok, reinterpret_cast<int*>(hist) + (tid >> 5) * E, t0, ra, rb, (long long)blockIdx.x + s);
      }
  }
  for (int k = 0; k < n_runs; ++k) {
    const int ra = PACKED ? runs.begin[k] : 0, rb = PACKED ? runs.begin[k + 1] : rows, s = PACKED ? runs.seq[ra] : 0;
    if (s < 0 || (n_runs > 1 && rb - ra < kWarpRows)) continue;
    for (int e = tid; e < E; e += kTileThreads) cnt[e] = 0;
    if (USAGE)
      for (int i = tid; i < kTileWarps * E; i += kTileThreads) hist[i] = 0.f;
    const int n = __syncthreads_count(tid >= ra && tid < rb && ok[min(tid, kMaxTileRows - 1)]);
    // choices: counts by integer atomics; the weights by rounds in which no two lanes of a warp hold the same expert,
    // each warp on a table of its own, so their sums have a fixed order
    const int i0 = ra * K, i1 = rb * K;
    for (int base = i0; base < i1; base += kTileThreads) {
      const int i = base + tid;
      int e = -1;
      if (i < i1 && ok[K == 1 ? i : (int)__umulhi((uint32_t)i, a.by_k)]) {
        const long long v = a.topi[t0 * K + i];
        if (v >= 0 && v < E) {
          e = (int)v;
          atomicAdd(&cnt[e], 1);
        } else {
          dev_fail(a.err, kDevErrBadIndex);
        }
      }
      if (USAGE) {
        float w = 0.f;
        if (e >= 0)
          w = a.topv_f32 ? reinterpret_cast<const float*>(a.topv)[t0 * K + i]
                         : __bfloat162float(reinterpret_cast<const bf16*>(a.topv)[t0 * K + i]);
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << (tid & 31)) - 1));
        const int rounds = __reduce_max_sync(0xffffffffu, e >= 0 ? rank + 1 : 0);
        float* h = hist + (tid >> 5) * E;
        for (int r = 0; r < rounds; ++r) {
          if (e >= 0 && rank == r) h[e] += w;
          __syncwarp();
        }
      }
    }
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (lane < lanes) {
      // U rows in flight; a row that does not count is read and left out (its values may be anything)
      constexpr int U = 4;
      const float* p = a.probs + t0 * a.ld + col;
      for (int r = ra + lane; r < rb; r += U * lanes) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int q = min(r + u * lanes, rb - 1);
          if constexpr (VEC == 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p + q * a.ld));
            v[u][0] = f.x;
            v[u][1] = f.y;
            v[u][2] = f.z;
            v[u][3] = f.w;
          } else {
            v[u][0] = __ldg(p + q * a.ld);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool counts = r + u * lanes < rb && ok[min(r + u * lanes, rb - 1)];
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += counts ? v[u][j] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[lane * ncol * VEC + col + j] = acc[j];
    }
    __syncthreads();
    const long long rec = (long long)blockIdx.x + s;
    for (int e = tid; e < E; e += kTileThreads) {
      float m = 0.f;
      for (int l = 0; l < lanes; ++l) m += red[l * ncol * VEC + e];
      a.rec_mass[rec * E + e] = m;
      a.rec_cnt[rec * E + e] = cnt[e];
      if (USAGE) {
        float w = 0.f;
        for (int l = 0; l < kTileWarps; ++l) w += hist[l * E + e];
        a.rec_weight[rec * E + e] = w;
      }
    }
    if (tid == 0) a.rec_n[rec] = n;
    __syncthreads();
  }
}

struct FinArgs {
  const float *rec_mass, *rec_weight;
  const int *rec_cnt, *rec_n;
  const int* cu;
  int S, E, K, rows;
  long long T;
  long long* counts;  // [S][E]
  float* coef;        // [S][E] gradient rows before the division by S', then [1] = 1 / S'
  float* loss;
  float *prob_mass, *weight_mass;  // usage
  double* part;       // [S][gridDim.y]
  int* seq_n;         // [S]
  int* ticket;
};

// The last block to finish adds the parts of the sequences (gridDim.y each) in their order.
__device__ __forceinline__ void finish_loss(const FinArgs& a) {
  constexpr int WARPS = kFinThreads / 32;
  __shared__ double sums[WARPS];
  __shared__ int somes[WARPS];
  __threadfence();
  const volatile double* parts = a.part;
  const volatile int* seqs = a.seq_n;
  double sum = 0.0;
  int some = 0;
  for (long long i = threadIdx.x; i < (long long)a.S * gridDim.y; i += kFinThreads) sum += parts[i];
  for (int i = threadIdx.x; i < a.S; i += kFinThreads) some += seqs[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    some += __shfl_xor_sync(0xffffffffu, some, o);
  }
  if (threadIdx.x % 32 == 0) {
    sums[threadIdx.x / 32] = sum;
    somes[threadIdx.x / 32] = some;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    some = 0;
    for (int l = 0; l < WARPS; ++l) {
      sum += sums[l];
      some += somes[l];
    }
    const double inv = 1.0 / max(some, 1);
    *a.loss = (float)(sum * inv);
    a.coef[(long long)a.S * a.E] = (float)inv;
  }
}

template <bool USAGE, int COLS>
__global__ void __launch_bounds__(kFinThreads) balance_finish_kernel(const FinArgs a) {
  constexpr int LANES = kFinThreads / COLS;
  __shared__ double sm[LANES][COLS + 1];
  __shared__ double sw[USAGE ? LANES : 1][COLS + 1];
  __shared__ int sc[LANES][COLS + 1];
  __shared__ int sn[LANES];
  __shared__ bool last;
  const int s = blockIdx.x, col = threadIdx.x % COLS, lane = threadIdx.x / COLS, E = a.E;
  const int e = blockIdx.y * COLS + col;
  long long lo, hi;
  seq_range(a.cu, s, a.T, lo, hi);
  double m = 0.0, w = 0.0;
  int c = 0, n = 0;
  if (lo < hi) {
    const int b1 = (int)((hi - 1) / a.rows);
#pragma unroll 4
    for (int b = (int)(lo / a.rows) + lane; b <= b1; b += LANES) {
      const long long rec = (long long)b + s;
      n += a.rec_n[rec];
      if (e < E) {
        m += a.rec_mass[rec * E + e];
        c += a.rec_cnt[rec * E + e];
        if (USAGE) w += a.rec_weight[rec * E + e];
      }
    }
  }
  sm[lane][col] = m;
  sc[lane][col] = c;
  if (USAGE) sw[lane][col] = w;
  if (col == 0) sn[lane] = n;
  __syncthreads();
  // the first warp adds the lanes' sums: 32 / COLS threads to a column, then across them
  if (threadIdx.x < 32) {
    m = w = 0.0;
    long long cs = 0, ns = 0;
#pragma unroll 8
    for (int l = lane; l < LANES; l += 32 / COLS) {
      m += sm[l][col];
      cs += sc[l][col];
      ns += sn[l];
      if (USAGE) w += sw[l][col];
    }
#pragma unroll
    for (int o = 16; o >= COLS; o >>= 1) {
      m += __shfl_xor_sync(0xffffffffu, m, o);
      cs += __shfl_xor_sync(0xffffffffu, cs, o);
      ns += __shfl_xor_sync(0xffffffffu, ns, o);
      if (USAGE) w += __shfl_xor_sync(0xffffffffu, w, o);
    }
    double part = 0.0;
    if (e < E && lane == 0) {
      a.counts[(long long)s * E + e] = cs;
      if (USAGE) {
        a.prob_mass[e] = (float)m;
        a.weight_mass[e] = (float)w;
      } else {
        const double f = ns ? (double)E * (double)cs / ((double)a.K * (double)ns * (double)ns) : 0.0;
        a.coef[(long long)s * E + e] = (float)f;
        part = f * m;
      }
    }
    if (!USAGE) {
#pragma unroll
      for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (threadIdx.x == 0) {
        a.part[(long long)s * gridDim.y + blockIdx.y] = part;
        if (blockIdx.y == 0) a.seq_n[s] = (int)min(ns, 1LL);
        __threadfence();
        last = atomicAdd(a.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1;
      }
    }
  }
  if (USAGE) return;
  __syncthreads();
  if (last) finish_loss(a);
}

// The same with a warp for 32 experts of a sequence, where sequences are short: at most a few records each.
__global__ void __launch_bounds__(kFinThreads) balance_finish_short_kernel(const FinArgs a) {
  __shared__ bool last;
  const int s = blockIdx.x * (kFinThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31, E = a.E;
  const int e = blockIdx.y * 32 + lane;
  if (s < a.S) {
    long long lo, hi;
    seq_range(a.cu, s, a.T, lo, hi);
    double m = 0.0;
    long long c = 0, n = 0;
    if (lo < hi) {
      const int b1 = (int)((hi - 1) / a.rows);
#pragma unroll 8
      for (int b = (int)(lo / a.rows); b <= b1; ++b) {
        const long long rec = (long long)b + s;
        n += a.rec_n[rec];
        if (e < E) {
          m += a.rec_mass[rec * E + e];
          c += a.rec_cnt[rec * E + e];
        }
      }
    }
    double part = 0.0;
    if (e < E) {
      const double f = n ? (double)E * (double)c / ((double)a.K * (double)n * (double)n) : 0.0;
      a.counts[(long long)s * E + e] = c;
      a.coef[(long long)s * E + e] = (float)f;
      part = f * m;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) {
      a.part[(long long)s * gridDim.y + blockIdx.y] = part;
      if (blockIdx.y == 0) a.seq_n[s] = n > 0;
      __threadfence();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1;
  __syncthreads();
  if (last) finish_loss(a);
}

// dprobs[t, :] = go / S' * coef[s(t), :] on the kept rows of the sequences, 0 elsewhere.
// Four roundings to fp32: of a coefficient, which is fp32 to halve what many sequences read, of 1 / S', which comes from another
// block, of go / S' and of the product. Products in fp64, formed once for a thread's rows of a sequence, leave two of them
// but took 0.2 to 1 us longer at every size measured.
template <int VEC>
__global__ void __launch_bounds__(kTileThreads)
    balance_bwd_kernel(const float* __restrict__ coef, const float* __restrict__ go, const uint8_t* __restrict__ mask,
                       const int* __restrict__ cu, int S, long long T, int E, int rows_per, float* __restrict__ dprobs) {
  __shared__ int seq[kMaxTileRows];
  const int tid = threadIdx.x;
  const long long t0 = (long long)blockIdx.x * rows_per;
  const int rows = (int)min((long long)rows_per, T - t0);
  const float g = *go * coef[(long long)S * E];
  int s0, s1;
  sequences_of(cu, S, t0, t0 + rows - 1, s0, s1);
  if (tid < rows) {
    const long long t = t0 + tid;
    seq[tid] = !mask || mask[t] ? sequence_of(cu, S, t, s0, s1) : -1;
  }
  __syncthreads();
  const int ncol = (E + VEC - 1) / VEC, lanes = kTileThreads / ncol;
  const int lane = tid / ncol, col = (tid - lane * ncol) * VEC;
  if (lane >= lanes) return;
#pragma unroll 4
  for (int r = lane; r < rows; r += lanes) {
    const int s = seq[r];
    float* d = dprobs + (t0 + r) * E + col;
    if (VEC == 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s >= 0) {
        v = *reinterpret_cast<const float4*>(coef + (long long)s * E + col);
        v = make_float4(v.x * g, v.y * g, v.z * g, v.w * g);
      }
      *reinterpret_cast<float4*>(d) = v;
    } else {
      *d = s >= 0 ? coef[(long long)s * E + col] * g : 0.f;
    }
  }
}

// Rows of a tile: enough tiles for four blocks on each of 148 SMs, at least 16 rows (a record costs as much traffic as
// two rows) and at most kMaxTileRows (the tile's flags, and the length of its fp32 sums).
int tile_rows(long long T) {
  const long long r = (T + 591) / 592;
  return (int)std::min<long long>(kMaxTileRows, std::max<long long>(16, (r + 15) / 16 * 16));
}

struct Layout {
  long long mass, weight, cnt, n, part, seq_n, ticket, total;
  int rows, tiles;
  int cols;  // experts of a finishing block (0: a warp for 32 experts of a sequence)
};

Layout layout(long long T, long long E, long long S, bool usage) {
  Layout l{};
  l.rows = tile_rows(T);
  l.tiles = (int)((T + l.rows - 1) / l.rows);
  l.cols = usage ? 8 : S > 16 && l.tiles < 4 * S ? 0 : S * E < 32 * 148 ? 8 : 32;
  const long long recs = l.tiles + S, eb = (E + 31) / 32 * (l.cols == 8 ? 4 : 1);
  long long o = 0;
  auto take = [&](long long bytes) {
    const long long at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  l.mass = take(recs * E * 4);
  l.weight = usage ? take(recs * E * 4) : 0;
  l.cnt = take(recs * E * 4);
  l.n = take(recs * 4);
  l.part = usage ? 0 : take(S * eb * 8);
  l.seq_n = usage ? 0 : take(S * 4);
  l.ticket = take(4);
  l.total = o;
  return l;
}

int check_sizes(const char* what, int64_t T, int64_t E, int64_t K, int64_t S) {
  SMELB_CHECK_ARG(T >= 0 && T < (1LL << 31) && E >= 1 && E <= kMaxE && K >= 1 && K <= kMaxK && S >= 1 && S < (1LL << 24),
                  kErrShape, "%s: T=%lld E=%lld K=%lld sequences=%lld", what, (long long)T, (long long)E, (long long)K,
                  (long long)S);
  return kOk;
}

// Factor of the division of a tile's choice by K.
uint32_t by(int64_t K) { return (uint32_t)((1ull << 32) / K + 1); }

template <bool USAGE>
int run_tiles(const TileArgs& t, int tiles, cudaStream_t st) {
  if (!tiles) return kOk;
  const bool vec = t.E % 4 == 0 && t.ld % 4 == 0 && ((uintptr_t)t.probs & 15) == 0;
  const size_t smem = USAGE || t.cu ? (size_t)kTileWarps * t.E * sizeof(float) : 0;
  constexpr int kAlone = USAGE ? kUsage : kOne, kSeqs = USAGE ? kUsage : kPacked;
  auto kern = t.cu ? (vec ? balance_tile_kernel<4, kSeqs> : balance_tile_kernel<1, kSeqs>)
                   : (vec ? balance_tile_kernel<4, kAlone> : balance_tile_kernel<1, kAlone>);
  kern<<<tiles, kTileThreads, smem, st>>>(t);
  SMELB_CUDA(cudaGetLastError());
  count_launch();
  return kOk;
}

template <bool USAGE>
int run_finish(const FinArgs& f, int cols, cudaStream_t st) {
  const dim3 grid((unsigned)f.S, (unsigned)((f.E + std::max(cols, 1) - 1) / std::max(cols, 1)));
  if (USAGE || cols == 8) {
    balance_finish_kernel<USAGE, 8><<<grid, kFinThreads, 0, st>>>(f);
  } else if (cols == 32) {
    balance_finish_kernel<false, 32><<<grid, kFinThreads, 0, st>>>(f);
  } else {
    const int per = kFinThreads / 32;
    balance_finish_short_kernel<<<dim3((unsigned)((f.S + per - 1) / per), (unsigned)((f.E + 31) / 32)), kFinThreads, 0,
                                  st>>>(f);
  }
  SMELB_CUDA(cudaGetLastError());
  count_launch();
  return kOk;
}

}  // namespace
}  // namespace smelb

using namespace smelb;

extern "C" {

int64_t smelb_balance_workspace_bytes(int64_t T, int64_t E, int64_t S, int usage) {
  if (T < 0 || E < 1 || S < 1) return 0;
  return layout(T, E, S, usage != 0).total;
}

int smelb_balance_loss_fwd(const float* probs, int64_t ld, const int64_t* topi, const uint8_t* mask,
                           const int32_t* cu_seqlens, int64_t S, int64_t T, int64_t E, int64_t K, float* loss,
                           int64_t* counts, float* coef, void* workspace, int64_t workspace_bytes, void* stream) {
  SMELB_CHECK_ARG((T == 0 || (probs && topi)) && loss && counts && coef && workspace, kErrArg,
                  "balance_loss_fwd: null pointer");
  if (int rc = check_sizes("balance_loss_fwd", T, E, K, S)) return rc;
  SMELB_CHECK_ARG(cu_seqlens || S == 1, kErrArg, "balance_loss_fwd: %lld sequences without cu_seqlens", (long long)S);
  SMELB_CHECK_ARG(ld >= E || T <= 1, kErrShape, "balance_loss_fwd: row pitch %lld for %lld experts", (long long)ld,
                  (long long)E);
  const Layout l = layout(T, E, S, false);
  SMELB_CHECK_ARG(workspace_bytes >= l.total, kErrWorkspace, "balance_loss_fwd: workspace %lld bytes, %lld needed",
                  (long long)workspace_bytes, l.total);
  SMELB_CHECK_ARG(((uintptr_t)workspace & 255) == 0, kErrArg, "balance_loss_fwd: workspace must be 256-byte aligned");
  int dev = 0;
  SMELB_CUDA(cudaGetDevice(&dev));
  char* ws = (char*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  int* ticket = (int*)(ws + l.ticket);
  if (l.tiles == 0) SMELB_CUDA(cudaMemsetAsync(ticket, 0, sizeof(int), st));
  const TileArgs t{probs, ld, (const long long*)topi, nullptr, 0, mask, cu_seqlens, (int)S, (int)E, (int)K, l.rows, by(K), T,
                   (float*)(ws + l.mass), nullptr, (int*)(ws + l.cnt), (int*)(ws + l.n), ticket,
                   device_status_on(dev, st)};
  if (int rc = run_tiles<false>(t, l.tiles, st)) return rc;
  const FinArgs f{t.rec_mass, nullptr, t.rec_cnt, t.rec_n, cu_seqlens, (int)S, (int)E, (int)K, l.rows, T,
                  (long long*)counts, coef, loss, nullptr, nullptr, (double*)(ws + l.part), (int*)(ws + l.seq_n),
                  ticket};
  return run_finish<false>(f, l.cols, st);
}

int smelb_balance_loss_bwd(const float* coef, const float* go, const uint8_t* mask, const int32_t* cu_seqlens,
                           int64_t S, int64_t T, int64_t E, float* dprobs, void* stream) {
  SMELB_CHECK_ARG(coef && go && (dprobs || T == 0), kErrArg, "balance_loss_bwd: null pointer");
  if (int rc = check_sizes("balance_loss_bwd", T, E, 1, S)) return rc;
  SMELB_CHECK_ARG(cu_seqlens || S == 1, kErrArg, "balance_loss_bwd: %lld sequences without cu_seqlens", (long long)S);
  if (T == 0) return kOk;
  cudaStream_t st = (cudaStream_t)stream;
  const int rows = tile_rows(T);
  const int tiles = (int)((T + rows - 1) / rows);
  const bool vec = E % 4 == 0 && (((uintptr_t)dprobs | (uintptr_t)coef) & 15) == 0;
  auto kern = vec ? balance_bwd_kernel<4> : balance_bwd_kernel<1>;
  kern<<<tiles, kTileThreads, 0, st>>>(coef, go, mask, cu_seqlens, (int)S, T, (int)E, rows, dprobs);
  SMELB_CUDA(cudaGetLastError());
  count_launch();
  return kOk;
}

int smelb_expert_usage(const float* probs, int64_t ld, const void* topv, int topv_fp32, const int64_t* topi,
                       const uint8_t* mask, int64_t T, int64_t E, int64_t K, int64_t* counts, float* prob_mass,
                       float* weight_mass, void* workspace, int64_t workspace_bytes, void* stream) {
  SMELB_CHECK_ARG((T == 0 || (probs && topi && topv)) && counts && prob_mass && weight_mass && workspace, kErrArg,
                  "expert_usage: null pointer");
  if (int rc = check_sizes("expert_usage", T, E, K, 1)) return rc;
  SMELB_CHECK_ARG(ld >= E || T <= 1, kErrShape, "expert_usage: row pitch %lld for %lld experts", (long long)ld,
                  (long long)E);
  const Layout l = layout(T, E, 1, true);
  SMELB_CHECK_ARG(workspace_bytes >= l.total, kErrWorkspace, "expert_usage: workspace %lld bytes, %lld needed",
                  (long long)workspace_bytes, l.total);
  SMELB_CHECK_ARG(((uintptr_t)workspace & 255) == 0, kErrArg, "expert_usage: workspace must be 256-byte aligned");
  int dev = 0;
  SMELB_CUDA(cudaGetDevice(&dev));
  char* ws = (char*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  const TileArgs t{probs, ld, (const long long*)topi, topv, topv_fp32, mask, nullptr, 1, (int)E, (int)K, l.rows, by(K), T,
                   (float*)(ws + l.mass), (float*)(ws + l.weight), (int*)(ws + l.cnt), (int*)(ws + l.n),
                   (int*)(ws + l.ticket), device_status_on(dev, st)};
  if (int rc = run_tiles<true>(t, l.tiles, st)) return rc;
  const FinArgs f{t.rec_mass, t.rec_weight, t.rec_cnt, t.rec_n, nullptr, 1, (int)E, (int)K, l.rows, T,
                  (long long*)counts, nullptr, nullptr, prob_mass, weight_mass, nullptr, nullptr, nullptr};
  return run_finish<true>(f, l.cols, st);
}

}  // extern "C"
